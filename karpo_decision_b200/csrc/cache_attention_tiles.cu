// Attention of new rows over cached e4m3 blocks for many query rows per key/value head (questions, chunks of prompts): the
// formulas and the visibility rule of cache_attention.cu, on the 5th-generation tensor cores.
//
// The rows of a request that share a key/value head (row r is token r / group, query head r % group of the head) are cut
// into tiles of 128, so a group's heads read the codes together. S = Q K^T and O += P V are tcgen05.mma with S, P and O in
// tensor memory, as in attention.cu; what differs is the operands. The keys' codes go to the tensor cores as they are
// (kind::f8f6f4, tiles by TMA): a query row is split into two e4m3 rows, its rounding and the rest, q 2^-e = hi + lo with
// the row's largest magnitude in (224, 448]. That is exact for every bf16 element within 2^-10 of the row's largest and
// off by at most 2^-10 (2^-17 of the largest) below, and two products at the 8-bit rate cost what one in 16 bits does. (The
// kernel for few rows holds queries in f16, 2^-25: a row with one large element may differ there in its last bits.)
// The values meet probabilities, which need more range than e4m3 has: converter warps load a block's value codes (16
// bytes a thread and piece, the next tile's loads in flight while one is converted, later tiles on their way into L2) and
// write them as f16 (exact, two per instruction) into the 128-byte swizzled tiles that the descriptors name. So the codes
// cross HBM and L2 as bytes. The blocks' scales never touch the elements: the key scale joins the softmax scale, the
// value scale the probabilities.
//
// Work is shared by weight, not by tile lists: every (request, key/value head, row tile, value slice) has a weight close
// to its visible keys whose prefix sums have a closed form, CTA c of P takes the c-th part of the total, and a part of an
// item takes its key tiles in proportion. So a few long items and many short ones keep every CTA equally busy without the
// host knowing a length. An item in one CTA's part is finished there; the others leave float32 partials (at most two per
// CTA) that a second launch joins.
//
// Warps: 0-3 softmax and epilogue, a thread a row (they also split the item's query rows), 4 work fetch and the keys' TMA
// loads, 5 MMA issue, 6.. conversion of values.
#include "cache_attention.cuh"

namespace kd {
namespace ct {

using namespace ca;

template <int HD, int DV>
struct Cfg {
  static constexpr int BM = 128;
  static constexpr int ROW = HD < 128 ? HD : 128;  // bytes of a key or query row within a swizzle chunk
  static constexpr int CHUNKS = HD / ROW;          // swizzle chunks along the head dim (Q, K)
  static constexpr int V_CHUNKS = DV / 64;         // 64 f16 values each
  static constexpr int SLICES = HD / DV;           // value slices, separate items
  static constexpr int Q_CHUNK = BM * ROW, K_CHUNK = BN * ROW, V_CHUNK = BN * 128;
  static constexpr int Q_BYTES = Q_CHUNK * CHUNKS;  // of hi, and of lo
  static constexpr int K_BYTES = K_CHUNK * CHUNKS;
  static constexpr int V_BYTES = V_CHUNK * V_CHUNKS;
  // Tensor-memory columns: O, NS score buffers (P overwrites its scores) and, for heads of 256, the queries (4 elements a
  // column): an A operand from shared memory costs 4 KB per 32 of head dim beside 2 KB of keys, more than the tensor core
  // waits for. Heads of 512 leave no room for them.
  static constexpr bool Q_TMEM = HD == 256;
  static constexpr int NS = HD == 64 ? 3 : HD == 512 ? 4 : 2;
  static constexpr int O_COL = 0, S_COL = DV, HI_COL = S_COL + NS * BN, LO_COL = HI_COL + HD / 4;
  // The order of the products: S_{j + 1} before P_j V_j, after a wait for the P V that read its buffer. (Scores queued
  // right behind P_j V_j without that wait took 3% off heads of 256, but only products into one accumulator are
  // documented to run in the order they were issued in.)
  static constexpr int USED_COLS = HI_COL + (Q_TMEM ? HD / 2 : 0), TMEM_COLS = USED_COLS <= 256 ? 256 : 512;
  static constexpr int QS_BYTES = Q_TMEM ? 0 : 2 * Q_BYTES;  // queries in shared memory
  static constexpr int KST = HD <= 128 ? 3 : HD == 256 ? 4 : 2, VST = HD <= 128 ? 3 : HD == 256 ? 4 : 1;  // ring stages
  static constexpr int TILES = QS_BYTES + KST * K_BYTES + VST * V_BYTES + (Q_TMEM ? BM * ROW : 0);  // of 1,024 bytes
  static constexpr int SMEM = TILES + 3 * 1024;
  static constexpr int CTAS_PER_SM = (2 * (SMEM + 1024) <= 227 * 1024 && 2 * TMEM_COLS <= 512) ? 2 : 1;
  static constexpr int SOFT = 4;  // softmax warps, a thread a row
  static constexpr int CONV_WARPS = HD <= 128 ? 2 : 4;
  static constexpr int CONV = 32 * CONV_WARPS;
  static constexpr int THREADS = 32 * (SOFT + 2) + CONV;
  static constexpr int PARTIAL = BM * (DV + 3);  // floats: O, then (m, M, l) per row
  static_assert(KST + NS <= 8, "the ring of tile infos");
  static_assert(USED_COLS <= 512, "tensor memory budget");
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
  // Registers per thread when two CTAs share the SM (256 threads at 128 each): the softmax warps take what the others
  // leave (128 x (168 + 88) = 256 x 128).
  static constexpr bool SPLIT_REGISTERS = CTAS_PER_SM == 2;
  static_assert(!SPLIT_REGISTERS || THREADS == 256, "two warpgroups");
};

constexpr float THRESHOLD = 4.0f;   // log2 units a row's maximum may grow before its sums are rescaled
constexpr float P_EXPONENT = 11.f, P_SCALE = 2048.f;  // f16 probabilities hold p * 2^11: at most 2^15 with the threshold
constexpr int ITEM_TILES = 4;       // an item's own cost (queries, epilogue) in key tiles
constexpr int MIN_TILES = 6;        // the least share of a CTA in key tiles: less costs more to join than it saves

// A request's row tiles and their weights w(j) = min(base + step j, cap) + own, in units of a key tile / group: the key
// tiles that row tile j sees, about, up to the window's width.
struct Shape {
  int q0, lq, lk, tiles;
  int64_t base, cap, own;
  int step;  // 0 or 2: 128 rows reach 128 / group keys further
  KD_DEVICE int64_t before(int64_t j) const {  // weight of the tiles before j
    const int64_t grow = base >= cap ? 0 : step == 0 ? j : min(j, (cap - base + 1) >> 1);
    return grow * base + step * (grow * (grow - 1) / 2) + (j - grow) * cap + j * own;
  }
};

KD_DEVICE Shape shape(const Args& a, int i) {
  const Request r = request(a, i);
  Shape s;
  s.q0 = r.q0;
  s.lq = r.lq;
  s.lk = r.lk;
  s.tiles = (int)(((int64_t)r.lq * a.group + 127) / 128);
  const int64_t g = a.group;
  s.cap = g * r.lk / BN;
  s.base = a.right < 0 ? s.cap : min(s.cap, (g * max(r.lk - r.lq + (int64_t)a.right, (int64_t)0) + 128) / BN);
  s.step = a.right < 0 ? 0 : 2;
  if (a.left >= 0) s.cap = min(s.cap, (g * ((int64_t)a.left + 1 + max(a.right, 0)) + 128) / BN);
  s.own = g * ITEM_TILES;
  return s;
}

// The CTAs that take part of a total weight.
KD_DEVICE int parts(int64_t total, int64_t group, int ctas) {
  return (int)min((int64_t)ctas, max((int64_t)1, quotient(total, group * MIN_TILES)));
}

// An item's place in the list request > key/value head > row tile > value slice, and its weight interval.
struct Item {
  int i, h, tile, slice;
  Shape s;
  int64_t begin, end;
};

// The item holding weight x of request i, whose own weights begin at `start`.
template <int SLICES>
KD_DEVICE void find(const Args& a, int i, int64_t start, int64_t x, Item& it) {
  it.i = i;
  it.s = shape(a, i);
  const int64_t head = it.s.before(it.s.tiles) * SLICES;
  it.h = (int)quotient(x - start, head);
  const int64_t y = x - start - it.h * head;
  int lo = 0, hi = it.s.tiles - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (it.s.before(mid) * SLICES <= y)
      lo = mid;
    else
      hi = mid - 1;
  }
  it.tile = lo;
  const int64_t b = it.s.before(lo), w = it.s.before(lo + 1) - b;
  it.slice = SLICES == 1 ? 0 : (int)quotient(y - b * SLICES, w);
  it.begin = start + it.h * head + b * SLICES + it.slice * w;
  it.end = it.begin + w;
}

// The next item of the list (it.end is its begin); false at the end.
template <int SLICES>
KD_DEVICE bool next(const Args& a, Item& it) {
  it.begin = it.end;
  if (++it.slice == SLICES) {
    it.slice = 0;
    if (++it.tile == it.s.tiles) {
      it.tile = 0;
      if (++it.h == a.hkv) {
        it.h = 0;
        do {
          if (++it.i >= a.n) return false;
          it.s = shape(a, it.i);
        } while (it.s.tiles == 0);
      }
    }
  }
  it.end = it.begin + it.s.before(it.tile + 1) - it.s.before(it.tile);
  return true;
}

// Key tiles [first, first + n) that any row of a row tile may see.
struct Tiles {
  int first, n;
};
KD_DEVICE Tiles visible(const Args& a, const Shape& s, int tile) {
  const int r0 = tile * 128, r1 = (int)min((int64_t)r0 + 127, (int64_t)s.lq * a.group - 1);
  const int off = s.lk - s.lq;
  int lo = 0, hi = s.lk - 1;
  if (a.left >= 0) lo = max(0, r0 / a.group + off - a.left);
  if (a.right >= 0) hi = min(hi, r1 / a.group + off + a.right);
  Tiles t;
  t.first = lo / BN;
  t.n = hi < lo ? 0 : hi / BN - t.first + 1;
  return t;
}

// The key tiles [t0, t1) of an item of weights [begin, end) with n tiles that the weights [x0, x1) take.
KD_DEVICE void portion(int64_t begin, int64_t end, int64_t x0, int64_t x1, int n, int& t0, int& t1) {
  const int64_t w = end - begin;
  t0 = x0 <= begin ? 0 : (int)quotient((x0 - begin) * n, w);
  t1 = x1 >= end ? n : (int)quotient((x1 - begin) * n, w);
}

// What the roles of a CTA need of its next part of an item.
struct Work {
  int q0, lq, lk, h, slice;
  int r0, rows;        // packed rows of the tile
  int first, n;        // its key tiles
  int i;               // the request, < 0: no more work
  int slot;            // the partial it leaves, < 0: it is the whole item
  int pad;
};

// An item that begins in a CTA's share and ends in a later one, for the joining launch. rows 0: none.
struct Split {
  int64_t begin, end, total;  // its weights, and the launch's
  int q0, h, slice, r0, rows, tiles, last, np;  // `last`: the CTA that finishes it
  uint32_t left;  // bit p: the p-th CTA from the beginning one leaves a partial; for the first 32
  int pad;
  // Whether the p-th CTA from CTA `first` has any of the item's key tiles.
  KD_DEVICE bool leaves(int first, int p) const {
    const int64_t x0 = quotient(total * (first + p), np), x1 = quotient(total * (first + p + 1), np);
    int t0, t1;
    portion(begin, end, max(x0, begin), min(x1, end), tiles, t0, t1);
    return t0 < t1;
  }
};

// block * heads + head of an item's tile j, < 0: absent. Roles look up 32 tiles at a time, one a lane.
KD_DEVICE int block_of(const Args& a, const Work& w, int j) {
  if (j >= w.n) return -1;
  const int id = a.table[(int64_t)w.i * a.ldt + w.first + j];
  return id >= 0 && id < a.blocks ? id * a.hkv + w.h : -1;
}

KD_DEVICE uint4 load_codes(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
KD_DEVICE void prefetch_block(const uint8_t* p, int bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// Shared-memory descriptor of a K-major tile of 8-bit elements in rows of ROW bytes with ROW-byte swizzling.
template <int ROW>
KD_DEVICE uint64_t kmajor_desc(uint32_t addr) {
  if constexpr (ROW == 128) {
    return sw128_kmajor_desc(addr);
  } else {
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)1u << 16;
    d |= (uint64_t)(512u >> 4) << 32;  // 8 rows x 64 B
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)4u << 61;           // 64-byte swizzle
    return d;
  }
}
// Offset of 16-byte piece c of row r in such a tile (chunks of `chunk` bytes).
template <int ROW>
KD_DEVICE int swizzled(int r, int c, int chunk) {
  if constexpr (ROW == 128) {
    return (c >> 3) * chunk + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  } else {
    return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  }
}

// D[tmem] (+)= A[tmem] * B[smem]^T, 8-bit float operands.
KD_DEVICE void mma_f8_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate));
}
KD_DEVICE void tmem_st4(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}

// What the softmax needs of a key tile.
struct Info {
  float k_scale, v_exp;
  int live;  // 0: the block is absent
  int pad;
};

// What a CTA's warps share beside the tiles.
template <int HD, int DV>
struct Shared {
  using C = Cfg<HD, DV>;
  uint64_t q_full, k_full[C::KST], v_full[C::VST], k_empty[C::KST], v_empty[C::VST];
  uint64_t s_full[C::NS], p_full[C::NS], pv_done[C::NS], item_full[2], item_empty[2], drained;
  int64_t warp[C::THREADS / 32], start;
  Work works[2];
  Info info[8];           // by key tile: at most KST + NS tiles are between their load and their softmax
  int req;
  uint32_t tmem_slot;
};

template <int HD, int DV>
__global__ void __launch_bounds__(Cfg<HD, DV>::THREADS, Cfg<HD, DV>::CTAS_PER_SM)
    row_tiles_kernel(const __grid_constant__ CUtensorMap map_k, Args a, const uint8_t* __restrict__ v_codes) {
  using C = Cfg<HD, DV>;
  constexpr int KST = C::KST, VST = C::VST, NS = C::NS, SL = C::SLICES, SOFT = C::SOFT;
  // Tiles first: nothing is declared static, so the dynamic area keeps its 1,024-byte alignment without slack.
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(a.status, KD_OK, KD_DEVICE_TIMEOUT);
    return;
  }
  uint8_t* s_q = smem;
  uint8_t* s_k = smem + C::QS_BYTES;
  uint8_t* s_v = s_k + KST * C::K_BYTES;
  uint8_t* s_stage = C::Q_TMEM ? s_v + VST * C::V_BYTES : s_q;  // the epilogue's, 128 rows of ROW bytes
  Shared<HD, DV>& sh = *reinterpret_cast<Shared<HD, DV>*>(smem + C::TILES);
  uint64_t &q_full = sh.q_full, *k_full = sh.k_full, *v_full = sh.v_full, *k_empty = sh.k_empty, *v_empty = sh.v_empty;
  uint64_t *s_full = sh.s_full, *p_full = sh.p_full, *pv_done = sh.pv_done;
  uint64_t *item_full = sh.item_full, *item_empty = sh.item_empty;
  Work* works = sh.works;
  Info* infos = sh.info;
  int64_t* s_warp = sh.warp;
  int64_t& s_start = sh.start;
  int& s_req = sh.req;
  uint32_t& tmem_slot = sh.tmem_slot;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&q_full, SOFT);
    mbar_init(&sh.drained, 1);
    for (int s = 0; s < KST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(&v_full[s], C::CONV_WARPS);
      mbar_init(&v_empty[s], 1);
    }
    for (int b = 0; b < NS; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 128);
      mbar_init(&pv_done[b], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&item_full[b], 1);
      mbar_init(&item_empty[b], SOFT + 1 + C::CONV_WARPS);
    }
    fence_barrier_init();
  }
  if (warp == SOFT + 1) {
    tmem_alloc(&tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  // ---- this CTA's share: a scan of the requests' weights for the total, then (a second scan if the requests outnumber
  // the threads) for the share's first request
  int64_t w_mine = 0, w_before = 0;
  // The sum past this chunk (-1 once bounds fall: they name rows twice, for CTAs at once, and such a launch has no work);
  // the thread's own weight and prefix.
  auto scan = [&](int i0, int64_t carry) -> int64_t {
    const int i = i0 + tid;
    w_mine = 0;
    bool falls = false;
    if (i < a.n) {
      falls = a.cu[i + 1] < a.cu[i];
      const Shape s = shape(a, i);
      w_mine = s.before(s.tiles) * SL * a.hkv;
    }
    int64_t x = w_mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t px = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += px;
    }
    if (lane == 31) s_warp[warp] = x;
    falls = __syncthreads_or(falls) || carry < 0;
    w_before = carry + x - w_mine;
#pragma unroll
    for (int v = 0; v < C::THREADS / 32; ++v) {
      if (v < warp) w_before += s_warp[v];
      carry += s_warp[v];
    }
    __syncthreads();
    return falls ? -1 : carry;
  };
  int64_t total = 0;
  for (int i0 = 0; i0 < a.n; i0 += C::THREADS) total = scan(i0, total);
  total = max(total, (int64_t)0);
  const int np = parts(total, a.group, gridDim.x);
  const int64_t share_lo = quotient(total * blockIdx.x, np);
  const int64_t share_hi = (int)blockIdx.x < np ? quotient(total * (blockIdx.x + 1), np) : 0;
  int64_t again = 0;
  for (int i0 = 0; i0 < a.n; i0 += C::THREADS) {
    if (a.n > C::THREADS) again = scan(i0, again);
    if (w_mine > 0 && share_lo >= w_before && share_lo < w_before + w_mine) {
      s_req = i0 + tid;
      s_start = w_before;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp >= SOFT) {
  if constexpr (C::SPLIT_REGISTERS) set_registers_down<88>();  // one instruction for the whole warpgroup
  if (warp == SOFT) {
    // ------------------------------------------------------------ work fetch, keys
    const int64_t lo = share_lo, hi = share_hi;
    Item it;
    bool more = lo < hi;
    if (more) find<SL>(a, s_req, s_start, lo, it);
    if (lane == 0) tma_prefetch_desc(&map_k);
    Split begun = {};
    uint32_t g = 0;  // key tiles so far
    bool ok = true;
    int64_t issued[KST];  // the last use of each stage that a copy was issued for
#pragma unroll
    for (int s = 0; s < KST; ++s) issued[s] = -1;
    for (uint32_t k = 0; ok; ++k) {
      Work w;
      w.i = -1;
      w.n = 0;
      while (more && it.begin < hi) {
        const Tiles v = visible(a, it.s, it.tile);
        const int64_t x0 = max(lo, it.begin), x1 = min(hi, it.end);
        int t0, t1;
        portion(it.begin, it.end, x0, x1, v.n, t0, t1);
        const bool whole = x0 == it.begin && x1 == it.end;
        if (it.end > hi) {
          begun = Split{it.begin, it.end, total, it.s.q0, it.h, it.slice, it.tile * 128,
                        (int)min((int64_t)128, (int64_t)it.s.lq * a.group - it.tile * 128), v.n, 0, np, 0, 0};
        }
        if (whole || t0 < t1) {
          w.q0 = it.s.q0;
          w.lq = it.s.lq;
          w.lk = it.s.lk;
          w.h = it.h;
          w.slice = it.slice;
          w.r0 = it.tile * 128;
          w.rows = (int)min((int64_t)128, (int64_t)it.s.lq * a.group - w.r0);
          w.first = v.first + t0;
          w.n = t1 - t0;
          w.i = it.i;
          // an item begun by an earlier CTA leaves this one's first partial, one begun here its second
          w.slot = whole ? -1 : 2 * (int)blockIdx.x + (it.begin < lo ? 0 : 1);
          more = next<SL>(a, it);
          break;
        }
        more = next<SL>(a, it);
      }
      if (lane == 0) {
        ok = mbar_wait(&item_empty[k & 1], ((k >> 1) & 1) ^ 1, a.status);
        if (ok) {
          works[k & 1] = w;
          mbar_arrive(&item_full[k & 1]);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok || w.i < 0) break;
      int z_next = block_of(a, w, lane), z_now = -1, ve_now = 0;
      float ks_now = 0.f;
      for (int j = 0; j < w.n && ok; ++j) {
        if ((j & 31) == 0) {
          z_now = z_next;
          ks_now = z_now >= 0 ? a.k_scale[z_now] : 0.f;
          ve_now = z_now >= 0 ? exponent_of(a.v_scale[z_now]) : 0;
          z_next = block_of(a, w, j + 32 + lane);
        }
        const int z = __shfl_sync(0xffffffffu, z_now, j & 31);
        const float ks = __shfl_sync(0xffffffffu, ks_now, j & 31);
        const int ve = __shfl_sync(0xffffffffu, ve_now, j & 31);
        const uint32_t G = g + j;
        const int st = G % KST;
        if (lane == 0) {
          ok = mbar_wait(&k_empty[st], ((G / KST) & 1) ^ 1, a.status);
          if (ok) {
            infos[G & 7] = Info{ks, (float)ve, z >= 0, 0};
            // an absent block's keys are masked: whatever the stage holds will do
            if (z >= 0) {
              issued[st] = G / KST;
              mbar_arrive_expect_tx(&k_full[st], C::K_BYTES);
              for (int c = 0; c < C::CHUNKS; ++c)
                tma_load_3d(&map_k, &k_full[st], s_k + st * C::K_BYTES + c * C::K_CHUNK, c * C::ROW, 0, z);
            } else {
              mbar_arrive(&k_full[st]);
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
      }
      g += w.n;
    }
    {
      // the item this CTA begins and the next ones finish, for the launch that joins them; share p holds weight y when
      // floor(p total / np) <= y
      Split* d = reinterpret_cast<Split*>(a.descs) + blockIdx.x;
      const bool split = lo < hi && begun.begin >= lo && begun.end > hi;
      if (split) {
        begun.last = (int)min((int64_t)np - 1, quotient(begun.end * np - 1, total));
        const bool leaves = lane <= begun.last - (int)blockIdx.x && begun.leaves(blockIdx.x, lane);
        begun.left = __ballot_sync(0xffffffffu, leaves);
      }
      if (lane == 0) {
        if (split)
          *d = begun;
        else
          d->rows = 0;
      }
    }
    if (lane == 0) {
      // wait (bounded) for the copies in flight: roles that gave up do not before the shared memory goes away
      const uint64_t start = globaltimer();
      for (int s = 0; s < KST; ++s)
        while (issued[s] >= 0 && !mbar_try_wait(smem_u32(&k_full[s]), (uint32_t)issued[s] & 1) &&
               globaltimer() - start < 1000000000ull) {
        }
    }
  } else if (warp == SOFT + 1) {
    // ------------------------------------------------------------ MMA issue
    if (elect_one()) {
      constexpr uint32_t idesc_s = mma_idesc(0, C::BM, BN);     // e4m3, K-major A and B
      constexpr uint32_t idesc_o = mma_idesc(0, C::BM, DV, 1);  // f16, A from TMEM, MN-major B (V)
      const uint32_t sq = smem_u32(s_q);
      uint32_t g = 0, nq = 0;  // key tiles and items so far
      for (uint32_t k = 0;; ++k) {
        if (!mbar_wait(&item_full[k & 1], (k >> 1) & 1, a.status)) goto gave_up;
        const int n = works[k & 1].n;
        const bool end = works[k & 1].i < 0;
        mbar_arrive(&item_empty[k & 1]);
        if (end) break;
        if (n == 0) continue;
        if (!mbar_wait(&q_full, nq & 1, a.status)) goto gave_up;
        ++nq;
        auto issue_s = [&](int j) -> bool {
          const uint32_t G = g + j;
          const int st = G % KST;
          if (G >= NS && !mbar_wait(&pv_done[G % NS], ((G - NS) / NS) & 1, a.status)) return false;
          if (!mbar_wait(&k_full[st], (G / KST) & 1, a.status)) return false;
          tc_fence_after();
          const uint32_t sk = smem_u32(s_k + st * C::K_BYTES);
          const uint32_t d = tmem + C::S_COL + (G % NS) * BN;
#pragma unroll
          for (int half = 0; half < 2; ++half)  // hi, then lo
#pragma unroll
            for (int kk = 0; kk < HD / 32; ++kk) {
              const int c = kk * 32 / C::ROW, w = kk * 32 % C::ROW;
              const uint64_t key = kmajor_desc<C::ROW>(sk + c * C::K_CHUNK + w);
              if constexpr (C::Q_TMEM)
                mma_f8_ts(d, tmem + (half ? C::LO_COL : C::HI_COL) + kk * 8, key, idesc_s, (half | kk) > 0);
              else
                mma_f8_ss(d, kmajor_desc<C::ROW>(sq + half * C::Q_BYTES + c * C::Q_CHUNK + w), key, idesc_s,
                          (half | kk) > 0);
            }
          mma_commit(&k_empty[st]);
          mma_commit(&s_full[G % NS]);
          return true;
        };
        if (!issue_s(0)) goto gave_up;
        for (int j = 0; j < n; ++j) {
          if (j + 1 < n && !issue_s(j + 1)) goto gave_up;
          const uint32_t G = g + j;
          const int st = G % VST;
          if (!mbar_wait(&p_full[G % NS], (G / NS) & 1, a.status)) goto gave_up;
          if (!mbar_wait(&v_full[st], (G / VST) & 1, a.status)) goto gave_up;
          tc_fence_after();
          const uint32_t sv = smem_u32(s_v + st * C::V_BYTES);
          const uint32_t p = tmem + C::S_COL + (G % NS) * BN;
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            mma_f16_ts(tmem + C::O_COL, p + kk * 8, sw128_mnmajor_desc(sv + kk * 2048, C::V_CHUNK), idesc_o,
                       (j | kk) != 0);
          mma_commit(&v_empty[st]);
          mma_commit(&pv_done[G % NS]);
        }
        g += n;
      }
    gave_up:
      // wait (bounded) for the products in flight: roles that gave up do not before the tiles and tensor memory go away
      mma_commit(&sh.drained);
      const uint64_t start = globaltimer();
      while (!mbar_try_wait(smem_u32(&sh.drained), 0) && globaltimer() - start < 1000000000ull) {
      }
    }
  } else {
    // ------------------------------------------------------------ conversion of value tiles
    // A warp's pass covers 8 rows x 64 columns: lanes 0-3 the four 16-code pieces of one row, lanes 4-7 of the next,
    // whose f16 pieces fall on the other banks (the swizzle flips with the row's parity). Every pass is a constant away
    // from the lane's first place.
    constexpr int CW = C::CONV_WARPS, VP = 8 * C::V_CHUNKS / CW;  // passes a warp
    constexpr int AHEAD = 6;                                      // tiles between L2 prefetch and use
    const int cw = warp - SOFT - 2;
    const int row0 = cw * 8 + (lane >> 2), quarter = lane & 3;
    const int from = row0 * HD + quarter * 16;
    const int to = row0 * 128, piece0 = ((2 * quarter) ^ (row0 & 7)) << 4, piece1 = ((2 * quarter + 1) ^ (row0 & 7)) << 4;
    uint4 vr[VP];
    uint32_t g = 0;
    for (uint32_t k = 0;; ++k) {
      if (!mbar_wait(&item_full[k & 1], (k >> 1) & 1, a.status)) goto done;
      const Work w = works[k & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[k & 1]);
      if (w.i < 0) break;
      if (w.n == 0) continue;
      int z_now = block_of(a, w, lane), z_next = block_of(a, w, 32 + lane);
      int batch = 0;  // the 32 tiles z_now holds
      auto id = [&](int j) {  // the block of tile j, in this batch or the next
        const int x = __shfl_sync(0xffffffffu, z_now, j & 31), y = __shfl_sync(0xffffffffu, z_next, j & 31);
        return j >= w.n ? -1 : (j >> 5) == batch ? x : y;
      };
      auto load_v = [&](int z, int keys) {  // keys: rows of the block that hold tokens; the rest may hold NaN codes
        const uint8_t* p = v_codes + (int64_t)max(z, 0) * (BN * HD) + w.slice * DV + from;
        if (z >= 0 && keys >= BN) {
#pragma unroll
          for (int s = 0; s < VP; ++s)
            vr[s] = load_codes(p + (s % (8 / CW)) * CW * 8 * HD + s / (8 / CW) * 64);
        } else {
#pragma unroll
          for (int s = 0; s < VP; ++s)
            vr[s] = z >= 0 && row0 + (s % (8 / CW)) * CW * 8 < keys
                        ? load_codes(p + (s % (8 / CW)) * CW * 8 * HD + s / (8 / CW) * 64)
                        : make_uint4(0, 0, 0, 0);
        }
      };
      const int last_key = w.lk - w.first * BN;  // keys from the item's first tile to the request's last token
      load_v(id(0), last_key);
      for (int j = 0; j < w.n; ++j) {
        if (j >= 32 && (j & 31) == 0) {
          z_now = z_next;
          ++batch;
          z_next = block_of(a, w, j + 32 + lane);
        }
        if (cw == 0) {
          const int z = id(j + AHEAD);
          if (lane == 0 && z >= 0) prefetch_block(v_codes + (int64_t)z * (BN * HD), BN * HD);
        }
        const int z1 = id(j + 1);
        const uint32_t G = g + j;
        const int st = G % VST;
        if (!mbar_wait(&v_empty[st], ((G / VST) & 1) ^ 1, a.status)) goto done;
        uint8_t* tile = s_v + st * C::V_BYTES + to;
#pragma unroll
        for (int s = 0; s < VP; ++s) {
          uint8_t* dst = tile + s / (8 / CW) * C::V_CHUNK + (s % (8 / CW)) * CW * 8 * 128;
          uint4 lo, hi;
          codes_to_f16(vr[s].x, lo.x, lo.y);
          codes_to_f16(vr[s].y, lo.z, lo.w);
          codes_to_f16(vr[s].z, hi.x, hi.y);
          codes_to_f16(vr[s].w, hi.z, hi.w);
          *reinterpret_cast<uint4*>(dst + piece0) = lo;
          *reinterpret_cast<uint4*>(dst + piece1) = hi;
        }
        load_v(z1, last_key - (j + 1) * BN);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
      }
      g += w.n;
    }
  }
  } else {
    if constexpr (C::SPLIT_REGISTERS) set_registers_up<168>();
    // ------------------------------------------------------------ queries, softmax, epilogue
    const int r = tid;  // the row within the tile = TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    uint32_t g = 0;
    for (uint32_t k = 0;; ++k) {
      if (!mbar_wait(&item_full[k & 1], (k >> 1) & 1, a.status)) goto done;
      const Work& w = works[k & 1];  // released after the epilogue: read again where it is needed
      if (w.i < 0) break;
      const int n = w.n;
      const bool live = r < w.rows, warp_live = warp * 32 < w.rows;
      float q_scale = 1.f;
      if (n > 0) {
        // The row's queries as hi + lo. The last item's products have read theirs: its last scores were waited for.
        if (warp_live) {
          const int gr = w.r0 + (live ? r : 0), tok = gr / a.group, head = w.h * a.group + gr - tok * a.group;
          constexpr int PIECES = HD / 8;  // 8-element pieces of the row
          constexpr int HELD = PIECES <= 16 ? PIECES : 16;
          const uint4* src =
              reinterpret_cast<const uint4*>(a.q + (int64_t)(w.q0 + tok) * a.ldq + (int64_t)head * HD);
          uint4 x[HELD];
          uint32_t top = 0;  // the largest magnitude as a bf16 pattern
#pragma unroll
          for (int c0 = PIECES - HELD; c0 >= 0; c0 -= HELD) {  // the first pieces last: they stay in registers
#pragma unroll
            for (int c = 0; c < HELD; ++c) x[c] = live ? src[c0 + c] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int c = 0; c < HELD; ++c) {
              const uint32_t v[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) top = max(top, max(v[e] & 0x7fffu, (v[e] >> 16) & 0x7fffu));
            }
          }
          // the least e with the largest magnitude within 448 = 1.75 * 2^8
          const int e = min(max((int)(top >> 7) - 127 - 8 + ((top & 0x7fu) > 0x60u ? 1 : 0), -120), 120);
          q_scale = pow2i(e);
          // An infinity or a NaN makes every element NaN: the row is NaN wherever it sees a key.
          const float inv = top >= 0x7f80u ? __int_as_float(0x7fffffff) : pow2i(-e);
#pragma unroll
          for (int c0 = 0; c0 < PIECES; c0 += HELD) {
            if (c0 > 0) {
#pragma unroll
              for (int c = 0; c < HELD; ++c) x[c] = live ? src[c0 + c] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int c = 0; c < HELD; c += 2) {
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint4 xv = x[c + y / 2];
                const float2 f = unpack_bf16x2(y & 1 ? xv.z : xv.x), h = unpack_bf16x2(y & 1 ? xv.w : xv.y);
                const float4 q4 = make_float4(f.x * inv, f.y * inv, h.x * inv, h.y * inv);
                hi[y] = e4m3_pair(q4.x, q4.y) | (e4m3_pair(q4.z, q4.w) << 16);
                uint32_t h0, h1;
                codes_to_f16(hi[y], h0, h1);
                const float2 b0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
                const float2 b1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                lo[y] = e4m3_pair(q4.x - b0.x, q4.y - b0.y) | (e4m3_pair(q4.z - b1.x, q4.w - b1.y) << 16);
              }
              const int piece = (c0 + c) / 2, at = swizzled<C::ROW>(r, piece, C::Q_CHUNK);
              if constexpr (C::Q_TMEM) {
                tmem_st4(lane_base + C::HI_COL + 4 * piece, hi);
                tmem_st4(lane_base + C::LO_COL + 4 * piece, lo);
              } else {
                *reinterpret_cast<uint4*>(s_q + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(s_q + C::Q_BYTES + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              }
            }
          }
          if constexpr (C::Q_TMEM) {
            tmem_st_wait();
            tc_fence_before();
          } else {
            fence_async_smem();
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full);  // rows of other warps hold anything: they are never read back
      }
      // The row's visible keys [key_lo, key_hi], from the item's first tile on, and the tiles [clear0, clear1) that every
      // row of the tile sees whole.
      int key_lo, key_hi, clear0 = 0, clear1;
      {
        const int off = w.lk - w.lq, first = w.first * BN;
        const int pos0 = w.r0 / a.group + off, pos1 = (w.r0 + w.rows - 1) / a.group + off;
        const int pos = (w.r0 + (live ? r : 0)) / a.group + off;
        key_lo = (a.left >= 0 ? max(pos - a.left, 0) : 0) - first;
        key_hi = (a.right >= 0 ? min(w.lk - 1, pos + a.right) : w.lk - 1) - first;
        const int end = a.right >= 0 ? min(w.lk, pos0 + a.right + 1) : w.lk;
        clear1 = end <= 0 ? 0 : end / BN - w.first;
        if (a.left >= 0) clear0 = (max(pos1 - a.left, 0) + BN - 1) / BN - w.first;
      }
      q_scale *= a.scale_log2;
      // running maxima in log2 units, possibly stale by the threshold: of x (the row sum's base) and of x + e_v (O's)
      float m = -INFINITY, big = -INFINITY, l = 0.f;
      float ve_max = -1000.f;  // the largest value exponent so far (the same for every row)
      // One key tile. GENERAL: some key is hidden from some row, the block is absent, or its value scale lies so far under
      // an earlier one's that a probability that counts could vanish beside a larger scaled one, so that the row sum takes
      // exponentials of its own. The other form has no selects and one exponential for both.
      auto tile = [&](auto general, int j, const Info& info) -> bool {
        constexpr bool GENERAL = decltype(general)::value;
        const uint32_t G = g + j;
        const float mul = score_factor(q_scale, info.k_scale), ve = info.v_exp;
        const uint32_t s_addr = lane_base + C::S_COL + (G % NS) * BN;
        float sv[BN];
        {
          uint32_t t0[32], t1[32];
          tmem_ld32(s_addr, t0);
          tmem_ld32(s_addr + 32, t1);
          tmem_ld_wait_regs(t0, t1);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            sv[e] = __uint_as_float(t0[e]);
            sv[32 + e] = __uint_as_float(t1[e]);
          }
        }
        if constexpr (GENERAL) {
          const int lo = info.live ? key_lo - j * BN : BN, hi = key_hi - j * BN;
#pragma unroll
          for (int e = 0; e < BN; ++e) sv[e] = (e >= lo && e <= hi) ? sv[e] : -INFINITY;
        }
        float mx[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) mx[e] = sv[e];
#pragma unroll
        for (int e = 8; e < BN; e += 2) mx[(e / 2) & 7] = max3(mx[(e / 2) & 7], sv[e], sv[e + 1]);
        const float mraw = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
        const float mt = GENERAL && mraw == -INFINITY ? -INFINITY : mraw * mul;
        const bool need = mt + ve > big + THRESHOLD;
        if (__any_sync(0xffffffffu, need)) {
          const float f = need ? fast_exp2(big - (mt + ve)) : 1.f;
          if (j > 0) {  // rows that saw nothing so far hold zeros
            if (!mbar_wait(&pv_done[(G - 1) % NS], ((G - 1) / NS) & 1, a.status)) return false;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < DV; c += 32) {
              uint32_t t[32];
              tmem_ld32(lane_base + C::O_COL + c, t);
              tmem_ld_wait_regs(t);
#pragma unroll
              for (int e = 0; e < 32; ++e) t[e] = __float_as_uint(__uint_as_float(t[e]) * f);
              tmem_st32(lane_base + C::O_COL + c, t);
            }
            tmem_st_wait();
          }
          if (need) big = mt + ve;
        }
        if (mt > m + THRESHOLD) {
          l *= fast_exp2(m - mt);
          m = mt;
        }
        uint32_t pk[BN / 2];
        float2 part[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
        const float2 mul2v = make_float2(mul, mul);
        if constexpr (!GENERAL) {
          // What goes to the tensor cores is 2^(x + e_v + 11 - M); its sum times 2^(M - e_v - 11 - m) is the row sum's part.
          const float shift = big - ve - P_EXPONENT;
          const float2 shift2 = make_float2(-shift, -shift);
#pragma unroll
          for (int e = 0; e < BN / 2; ++e) {
            const float2 x = fma2(make_float2(sv[2 * e], sv[2 * e + 1]), mul2v, shift2);
            const float2 p = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            part[e & 3] = add2(part[e & 3], p);
            pk[e] = pack_f16x2(p.x, p.y);
          }
          const float2 ps = add2(add2(part[0], part[1]), add2(part[2], part[3]));
          l += (ps.x + ps.y) * fast_exp2(shift - m);
        } else {
          const float base = m == -INFINITY ? 0.f : m, vbase = big == -INFINITY ? 0.f : big;
          const float2 base2 = make_float2(-base, -base);
          const float factor = fast_exp2(fminf(base - vbase + ve + P_EXPONENT, 126.f));
#pragma unroll
          for (int e = 0; e < BN / 2; ++e) {
            const float2 x = fma2(make_float2(sv[2 * e], sv[2 * e + 1]), mul2v, base2);
            const float2 p = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            part[e & 3] = add2(part[e & 3], p);
            pk[e] = pack_f16x2(p.x * factor, p.y * factor);
          }
          const float2 ps = add2(add2(part[0], part[1]), add2(part[2], part[3]));
          l += ps.x + ps.y;
        }
        tmem_st32(s_addr, pk);
        tmem_st_wait();
        tc_fence_before();
        return true;
      };
      for (int j = 0; j < n; ++j) {
        const uint32_t G = g + j;
        if (!mbar_wait(&s_full[G % NS], (G / NS) & 1, a.status)) goto done;
        if (warp_live) {  // else no row of this warp: its probabilities are never read back
          tc_fence_after();
          const Info info = infos[G & 7];
          const bool ok = j < clear0 || j >= clear1 || !info.live || ve_max - info.v_exp > 80.f
                              ? tile(std::true_type{}, j, info)
                              : tile(std::false_type{}, j, info);
          if (!ok) goto done;
          ve_max = fmaxf(ve_max, info.v_exp);
        }
        mbar_arrive(&p_full[G % NS]);
      }
      // ---- epilogue
      if (n > 0) {
        const uint32_t G = g + n - 1;
        if (!mbar_wait(&pv_done[G % NS], (G / NS) & 1, a.status)) goto done;
        tc_fence_after();
      }
      if (warp_live) {
        const float base = m == -INFINITY ? 0.f : m, vbase = big == -INFINITY ? 0.f : big;
        const int gr = w.r0 + (live ? r : 0), tok = gr / a.group, head = w.h * a.group + gr - tok * a.group;
        const uint32_t o_addr = lane_base + C::O_COL;
        if (w.slot < 0) {
          // Through the warp's staging area (its rows' first chunk of the query tile, read by now), CC columns at a time:
          // the gate's rows in and the output's rows out as whole lines, ROW bytes of a row by ROW / 16 lanes.
          constexpr int CC = C::ROW / 2, LPR = C::ROW / 16, RPP = 32 / LPR;
          uint8_t* stage = s_stage + warp * 32 * C::ROW;
          const int piece = lane % LPR, sub = lane / LPR;
          const int64_t at = (int64_t)head * HD + w.slice * DV;
          const int64_t orow = (int64_t)(w.q0 + tok) * a.ldo + at, grow = (int64_t)(w.q0 + tok) * a.ldg + at;
          const float fin = l == 0.f ? 0.f : fast_exp2(fminf(vbase - base, 126.f)) / (l * P_SCALE);
#pragma unroll 1
          for (int c = 0; c < DV; c += CC) {
            if (a.gate) {
              uint4 gv[LPR];
#pragma unroll
              for (int p = 0; p < LPR; ++p) {
                const int rr = p * RPP + sub;
                const int64_t from = __shfl_sync(0xffffffffu, grow, rr) + c + piece * 8;
                gv[p] = warp * 32 + rr < w.rows ? *reinterpret_cast<const uint4*>(a.gate + from) : make_uint4(0, 0, 0, 0);
              }
#pragma unroll
              for (int p = 0; p < LPR; ++p)
                *reinterpret_cast<uint4*>(stage + swizzled<C::ROW>(p * RPP + sub, piece, 0)) = gv[p];
              __syncwarp();
            }
#pragma unroll
            for (int c2 = 0; c2 < CC; c2 += 32) {
              uint32_t t[32];
              if (n > 0) {
                tmem_ld32(o_addr + c + c2, t);
                tmem_ld_wait_regs(t);
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint4* mine = reinterpret_cast<uint4*>(stage + swizzled<C::ROW>(lane, c2 / 8 + q, 0));
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = l == 0.f ? 0.f : __uint_as_float(t[8 * q + e]) * fin;
                if (a.gate && l != 0.f) {
                  const uint4 gq = *mine;
                  const uint32_t gw[4] = {gq.x, gq.y, gq.z, gq.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float2 s = unpack_bf16x2(gw[e]);
                    x[2 * e] = x_sigmoid(x[2 * e], s.x);
                    x[2 * e + 1] = x_sigmoid(x[2 * e + 1], s.y);
                  }
                }
                *mine = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                   pack_bf16x2(x[6], x[7]));
              }
            }
            __syncwarp();
#pragma unroll
            for (int p = 0; p < LPR; ++p) {
              const int rr = p * RPP + sub;
              const int64_t to = __shfl_sync(0xffffffffu, orow, rr) + c + piece * 8;
              const uint4 y = *reinterpret_cast<const uint4*>(stage + swizzled<C::ROW>(rr, piece, 0));
              if (warp * 32 + rr < w.rows) *reinterpret_cast<uint4*>(a.out + to) = y;
            }
            __syncwarp();
          }
        } else {
          // [DV / 4][128 rows][4]: a warp's stores are whole lines; then m, M and l per row
          float* part = a.partials + (int64_t)w.slot * C::PARTIAL;
          if (live) {
            part[C::BM * DV + r] = m;
            part[C::BM * DV + 128 + r] = big;
            part[C::BM * DV + 256 + r] = l;
          }
#pragma unroll 1
          for (int c = 0; c < DV; c += 32) {
            uint32_t t[32];
            __syncwarp();
            tmem_ld32(o_addr + c, t);
            tmem_ld_wait_regs(t);
            if (live) {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                *reinterpret_cast<uint4*>(part + ((c / 4 + q) * 128 + r) * 4) =
                    make_uint4(t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3]);
            }
          }
        }
        // the next item's first product overwrites O: every row of this warp has read it
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[k & 1]);
      g += n;
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == SOFT + 1) {
    __syncwarp();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Joins the partials of the item that CTA blockIdx.x began and later ones finished, 8 of its 128 rows a block, a thread 4
// columns of a row. Up to JOIN_FEW partials (what a pack of requests leaves): every thread reads its row's statistics and
// its columns of four partials at once, in key order, with a running maximum; nothing waits for another thread, and the
// beginning CTA has worked out which shares hold tiles (8 requests of 20 to 200 rows: 162 -> 150 us with it). More (one
// long state): the statistics first, shared out among the threads, to a weight for each partial, then the columns, eight
// loads in flight.
constexpr int JOIN_MOST = 320;  // partials of an item: at most the CTAs
constexpr int JOIN_FEW = 16;
template <int HD, int DV>
__global__ void __launch_bounds__(2 * DV) join_tiles_kernel(Args a) {
  using C = Cfg<HD, DV>;
  constexpr int GROUPS = 2 * DV / 8;  // threads that share a row
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the partials are there after this
  const Split it = reinterpret_cast<const Split*>(a.descs)[blockIdx.x];
  if ((int)blockIdx.y * 8 >= it.rows) return;
  const int first = blockIdx.x, n = it.last - first + 1;
  const int sub = threadIdx.x & 7, c4 = threadIdx.x >> 3, r = blockIdx.y * 8 + sub;
  const bool live = r < it.rows;
  const int gr = it.r0 + r, tok = gr / a.group;
  const int64_t row = it.q0 + tok, col = (int64_t)(it.h * a.group + gr - tok * a.group) * HD + it.slice * DV + 4 * c4;
  uint2 gate = make_uint2(0, 0);
  if (a.gate && live) gate = *reinterpret_cast<const uint2*>(a.gate + row * a.ldg + col);
  float m = -INFINITY, big = -INFINITY, l = 0.f, base = 0.f, vbase = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (n <= JOIN_FEW) {
    for (int p0 = 0; p0 < n; p0 += 4) {
      float x[4], y[4], z[4];
      float4 v[4];
      float mm = m, bb = big;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        x[q] = y[q] = -INFINITY;
        z[q] = 0.f;
        v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (((it.left >> (p0 + q)) & 1u) && live) {
          const float* part = a.partials + (int64_t)(2 * (first + p0 + q) + (p0 + q == 0 ? 1 : 0)) * C::PARTIAL;
          const float* st = part + C::BM * DV + r;
          x[q] = st[0];
          y[q] = st[128];
          z[q] = st[256];
          v[q] = *reinterpret_cast<const float4*>(part + (c4 * 128 + r) * 4);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        mm = fmaxf(mm, x[q]);
        bb = fmaxf(bb, y[q]);
      }
      base = mm == -INFINITY ? 0.f : mm;
      vbase = bb == -INFINITY ? 0.f : bb;
      l *= fast_exp2(m - base);
      const float f = fast_exp2(big - vbase);
      o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
      m = mm;
      big = bb;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        l += z[q] * fast_exp2(x[q] - base);
        const float w = fast_exp2(y[q] - vbase);
        if (y[q] != -INFINITY || z[q] != 0.f) {  // otherwise no key of the row: its sums may hold anything
          o.x += v[q].x * w;
          o.y += v[q].y * w;
          o.z += v[q].z * w;
          o.w += v[q].w * w;
        }
      }
    }
    if (!live) return;
  } else {
    __shared__ float s_w[JOIN_MOST][8];
    __shared__ float s_red[3][2 * DV / 32][8];
    __shared__ int s_slot[JOIN_MOST];  // < 0: the share holds none of the item's tiles
    for (int p = threadIdx.x; p < n; p += 2 * DV) s_slot[p] = it.leaves(first, p) ? 2 * (first + p) + (p == 0 ? 1 : 0) : -1;
    __syncthreads();
    for (int p = c4; p < n; p += GROUPS) {
      const int slot = s_slot[p];
      if (slot < 0 || !live) continue;
      const float* st = a.partials + (int64_t)slot * C::PARTIAL + C::BM * DV + r;
      m = fmaxf(m, st[0]);
      big = fmaxf(big, st[128]);
    }
    auto across = [&](float v, int which, auto op) -> float {  // over the threads of a row
      v = op(v, __shfl_xor_sync(0xffffffffu, v, 8));
      v = op(v, __shfl_xor_sync(0xffffffffu, v, 16));
      if ((threadIdx.x & 31) < 8) s_red[which][threadIdx.x / 32][sub] = v;
      __syncthreads();
      v = s_red[which][0][sub];
#pragma unroll
      for (int q = 1; q < 2 * DV / 32; ++q) v = op(v, s_red[which][q][sub]);
      return v;
    };
    m = across(m, 0, [](float x, float y) { return fmaxf(x, y); });
    big = across(big, 1, [](float x, float y) { return fmaxf(x, y); });
    base = m == -INFINITY ? 0.f : m;
    vbase = big == -INFINITY ? 0.f : big;
    for (int p = c4; p < n; p += GROUPS) {
      const int slot = s_slot[p];
      float f = -1.f;
      if (slot >= 0 && live) {
        const float* st = a.partials + (int64_t)slot * C::PARTIAL + C::BM * DV + r;
        l += st[256] * fast_exp2(st[0] - base);
        if (st[128] != -INFINITY || st[256] != 0.f) f = fast_exp2(st[128] - vbase);
      }
      s_w[p][sub] = f;  // < 0: no key of the row (its sums may hold anything)
    }
    l = across(l, 2, [](float x, float y) { return x + y; });
    if (!live) return;
    for (int p0 = 0; p0 < n; p0 += 8) {
      float4 y[8];
      float f[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        f[q] = p0 + q < n ? s_w[p0 + q][sub] : -1.f;
        y[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (f[q] >= 0.f || f[q] != f[q])
          y[q] = *reinterpret_cast<const float4*>(a.partials + (int64_t)s_slot[p0 + q] * C::PARTIAL + (c4 * 128 + r) * 4);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float w = f[q] < 0.f ? 0.f : f[q];
        o.x += y[q].x * w;
        o.y += y[q].y * w;
        o.z += y[q].z * w;
        o.w += y[q].w * w;
      }
    }
  }
  const float fin = l == 0.f ? 0.f : fast_exp2(fminf(vbase - base, 126.f)) / (l * P_SCALE);
  float x[4] = {o.x * fin, o.y * fin, o.z * fin, o.w * fin};
  if (l == 0.f) {
    x[0] = x[1] = x[2] = x[3] = 0.f;
  } else if (a.gate) {
    const float2 s0 = unpack_bf16x2(gate.x), s1 = unpack_bf16x2(gate.y);
    x[0] = x_sigmoid(x[0], s0.x);
    x[1] = x_sigmoid(x[1], s0.y);
    x[2] = x_sigmoid(x[2], s1.x);
    x[3] = x_sigmoid(x[3], s1.y);
  }
  *reinterpret_cast<uint2*>(a.out + row * a.ldo + col) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
}

// Scratch: a Split per CTA, two partials per CTA.
static int64_t header_bytes(int ctas) { return ((int64_t)ctas * sizeof(Split) + 15) / 16 * 16; }

template <int HD, int DV>
int64_t workspace(int sms) {
  using C = Cfg<HD, DV>;
  const int64_t ctas = (int64_t)sms * C::CTAS_PER_SM;
  return header_bytes((int)ctas) + 2 * ctas * C::PARTIAL * (int64_t)sizeof(float);
}

template <int HD, int DV>
int launch(Args a, const void* k_codes, const uint8_t* v_codes, uint8_t* ws, int64_t ws_bytes, cudaStream_t stream) {
  using C = Cfg<HD, DV>;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(KD_ERR_ARGUMENT, "attention_cache: device index");
  const int sms = num_sms(dev), ctas = min(sms * C::CTAS_PER_SM, JOIN_MOST);
  if (ws_bytes < workspace<HD, DV>(sms))
    return set_error(KD_ERR_ARGUMENT, "attention_cache: workspace smaller than kd_attention_cache_workspace");
  a.descs = ws;
  a.partials = reinterpret_cast<float*>(ws + header_bytes(ctas));
  static_assert(sizeof(Shared<HD, DV>) <= C::SMEM - C::TILES, "shared memory layout");
  auto kernel = row_tiles_kernel<HD, DV>;
  static bool configured[64] = {false};
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return record_cuda_error(e, "attention_cache: cudaFuncSetAttribute");
    configured[dev] = true;
  }
  CUtensorMap mk;
  const auto sw = C::ROW == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  if (int rc = make_tma_3d(&mk, k_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, HD, BN, (uint64_t)a.blocks * a.hkv, HD,
                           (uint64_t)BN * HD, C::ROW, BN, 1, sw))
    return rc;
  kernel<<<ctas, C::THREADS, C::SMEM, stream>>>(mk, a, v_codes);
  if (int rc = record_cuda_error(cudaGetLastError(), "attention_cache: launch")) return rc;
  return launch_after(join_tiles_kernel<HD, DV>, dim3(ctas, 16), 2 * DV, stream, a);
}

}  // namespace ct

namespace ca {

int64_t row_tiles_workspace(int head_dim, int sms) {
  switch (head_dim) {
    case 64: return ct::workspace<64, 64>(sms);
    case 128: return ct::workspace<128, 128>(sms);
    case 256: return ct::workspace<256, 256>(sms);
    default: return ct::workspace<512, 256>(sms);
  }
}

int row_tiles(int head_dim, const Args& a, const void* k_codes, const void* v_codes, uint8_t* ws, int64_t ws_bytes,
              cudaStream_t stream) {
  const uint8_t* v = static_cast<const uint8_t*>(v_codes);
  switch (head_dim) {
    case 64: return ct::launch<64, 64>(a, k_codes, v, ws, ws_bytes, stream);
    case 128: return ct::launch<128, 128>(a, k_codes, v, ws, ws_bytes, stream);
    case 256: return ct::launch<256, 256>(a, k_codes, v, ws, ws_bytes, stream);
    default: return ct::launch<512, 256>(a, k_codes, v, ws, ws_bytes, stream);
  }
}

}  // namespace ca
}  // namespace kd
