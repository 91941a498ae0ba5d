// Attention of new rows over cached e4m3 blocks for many query rows per key/value head (questions, chunks of prompts): the
// formulas and the visibility rule of cache_attention.cu, on the 5th-generation tensor cores.
//
// The rows of a request that share a key/value head (row r is token r / group, query head r % group of the head) are cut
// into tiles of 128, so a group's heads read the codes together. S = Q K^T and O += P V are tcgen05.mma with S, P and O in
// tensor memory, as in attention.cu; what differs is the operands. The keys' codes go to the tensor cores as they are
// (kind::f8f6f4, tiles by TMA): a query row is split into two e4m3 rows, its rounding and the rest, q 2^-e = hi + lo with
// the row's largest magnitude in (224, 448]. That is exact for every bf16 element within 2^-10 of the row's largest and
// off by at most 2^-10 (2^-18 of the largest) below, and two products at the 8-bit rate cost what one in 16 bits does.
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
// Warps: 0-3 softmax and epilogue (one row a thread: its TMEM lane; they also split the item's query rows), 4 work fetch
// and the keys' TMA loads, 5 MMA issue, 6.. conversion of values.
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
  static constexpr int KST = HD <= 256 ? 3 : 2, VST = HD <= 256 ? 3 : 1;  // ring stages
  static constexpr int SMEM = 2 * Q_BYTES + KST * K_BYTES + VST * V_BYTES + 1024;
  static constexpr int O_COL = 0, S_COL = DV;
  static constexpr int TMEM_COLS = DV + 2 * BN <= 256 ? 256 : 512;
  static constexpr int NS = (TMEM_COLS - DV) / BN < 4 ? (TMEM_COLS - DV) / BN : 4;  // score buffers
  static constexpr int CTAS_PER_SM = (2 * (SMEM + 2048) <= 227 * 1024 && 2 * TMEM_COLS <= 512) ? 2 : 1;
  static constexpr int CONV_WARPS = HD <= 128 ? 2 : 4;
  static constexpr int CONV = 32 * CONV_WARPS;
  static constexpr int THREADS = 192 + CONV;
  static constexpr int PARTIAL = BM * (DV + 3);  // floats: O, then (m, M, l) per row
  static_assert(NS >= 2 && S_COL + NS * BN <= TMEM_COLS, "tensor memory budget");
  static_assert(SMEM + 1024 <= 227 * 1024, "shared memory budget");
  // Registers per thread when two CTAs share the SM (256 threads at 128 each): the softmax warps take what the others
  // leave (4 x 32 x (168 + 88) = 256 x 128).
  static constexpr bool SPLIT_REGISTERS = CTAS_PER_SM == 2;
  static_assert(!SPLIT_REGISTERS || THREADS == 256, "two warpgroups");
};

constexpr float THRESHOLD = 4.0f;   // log2 units a row's maximum may grow before its sums are rescaled
constexpr float P_SCALE = 2048.f;   // f16 probabilities hold p * 2^11: at most 2^15 with the threshold
constexpr int ITEM_TILES = 4;       // an item's own cost (queries, epilogue) in key tiles
constexpr int MIN_TILES = 6;        // the least share of a CTA in key tiles: less costs more to join than it saves

// A request's row tiles and their weights w(j) = min(base + step j, cap) + own (units: keys x group): the keys tile j
// sees, up to the window's width.
struct Shape {
  int q0, lq, lk, tiles;
  int64_t base, step, cap, own;
  KD_DEVICE int64_t before(int64_t j) const {  // weight of the tiles before j
    const int64_t grow = base >= cap ? 0 : step == 0 ? j : min(j, (cap - base + step - 1) / step);
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
  s.cap = g * r.lk;
  s.base = a.right < 0 ? s.cap : min(s.cap, g * max(r.lk - r.lq + (int64_t)a.right, (int64_t)0) + 128);
  s.step = a.right < 0 ? 0 : 128;
  if (a.left >= 0) s.cap = min(s.cap, g * ((int64_t)a.left + 1 + max(a.right, 0)) + 128);
  s.own = g * BN * ITEM_TILES;
  return s;
}

// The CTAs that take part of a total weight.
KD_DEVICE int parts(int64_t total, int64_t group, int ctas) {
  return (int)min((int64_t)ctas, max((int64_t)1, total / (group * BN * MIN_TILES)));
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
  it.h = (int)((x - start) / head);
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
  it.slice = (int)((y - b * SLICES) / w);
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

// The key tiles [t0, t1) of an item with n tiles that the weights [x0, x1) take.
KD_DEVICE void portion(const Item& it, int64_t x0, int64_t x1, int n, int& t0, int& t1) {
  const int64_t w = it.end - it.begin;
  t0 = x0 <= it.begin ? 0 : (int)((x0 - it.begin) * n / w);
  t1 = x1 >= it.end ? n : (int)((x1 - it.begin) * n / w);
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

// One tile's block and scales, looked up 32 tiles at a time by a warp's lanes.
struct Lookup {
  int z;  // block * heads + head, < 0: absent
  float k_scale;
  int v_exp;
};
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

template <int N>
KD_DEVICE void set_registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
KD_DEVICE void set_registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int HD, int DV>
__global__ void __launch_bounds__(Cfg<HD, DV>::THREADS, Cfg<HD, DV>::CTAS_PER_SM)
    row_tiles_kernel(const __grid_constant__ CUtensorMap map_k, Args a, const uint8_t* __restrict__ v_codes) {
  using C = Cfg<HD, DV>;
  constexpr int KST = C::KST, VST = C::VST, NS = C::NS, SL = C::SLICES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  uint8_t* s_k = smem + 2 * C::Q_BYTES;
  uint8_t* s_v = s_k + KST * C::K_BYTES;
  __shared__ uint64_t q_full, k_full[KST], v_full[VST], k_empty[KST], v_empty[VST], s_full[NS], p_full[NS], pv_done[NS];
  __shared__ uint64_t item_full[2], item_empty[2];
  __shared__ Work works[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int64_t s_warp[C::THREADS / 32], s_lo, s_hi, s_start;
  __shared__ int s_req;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&q_full, 128);
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
      mbar_init(&item_empty[b], 5 + C::CONV_WARPS);
    }
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(&tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  // ---- this CTA's share: a scan of the requests' weights, first for the total, then for the share's first request
  int64_t total = 0;
  int np = 1;
  for (int pass = 0; pass < 2; ++pass) {
    np = parts(total, a.group, gridDim.x);
    const int64_t lo = pass ? total * blockIdx.x / np : 0;
    int64_t carry = 0;
    for (int i0 = 0; i0 < a.n; i0 += C::THREADS) {
      const int i = i0 + tid;
      int64_t w = 0;
      if (i < a.n) {
        const Shape s = shape(a, i);
        w = s.before(s.tiles) * SL * a.hkv;
      }
      int64_t x = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t px = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += px;
      }
      if (lane == 31) s_warp[warp] = x;
      __syncthreads();
      int64_t before = carry, chunk = 0;
#pragma unroll
      for (int v = 0; v < C::THREADS / 32; ++v) {
        if (v < warp) before += s_warp[v];
        chunk += s_warp[v];
      }
      before += x - w;
      if (pass && i < a.n) {
        if (blockIdx.x == 0) a.tile_cu[i] = before;  // for the launch that joins the partials
        if (w > 0 && lo >= before && lo < before + w) {
          s_req = i;
          s_start = before;
        }
      }
      carry += chunk;
      __syncthreads();
    }
    total = carry;
    if (pass && tid == 0) {
      s_lo = lo;
      s_hi = (int)blockIdx.x < np ? total * (blockIdx.x + 1) / np : 0;
      if (blockIdx.x == 0) a.tile_cu[a.n] = total;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp >= 4) {
  if constexpr (C::SPLIT_REGISTERS) set_registers_down<88>();  // one instruction for the whole warpgroup
  if (warp == 4) {
    // ------------------------------------------------------------ work fetch, keys
    const int64_t lo = s_lo, hi = s_hi;
    Item it;
    bool more = lo < hi;
    if (more) find<SL>(a, s_req, s_start, lo, it);
    if (lane == 0) tma_prefetch_desc(&map_k);
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
        portion(it, x0, x1, v.n, t0, t1);
        const bool whole = x0 == it.begin && x1 == it.end;
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
      int z_next = block_of(a, w, lane), z_now = -1;
      for (int j = 0; j < w.n && ok; ++j) {
        if ((j & 31) == 0) {
          z_now = z_next;
          z_next = block_of(a, w, j + 32 + lane);
        }
        const int z = __shfl_sync(0xffffffffu, z_now, j & 31);
        const uint32_t G = g + j;
        const int st = G % KST;
        if (lane == 0) {
          ok = mbar_wait(&k_empty[st], ((G / KST) & 1) ^ 1, a.status);
          if (ok) {
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
    if (!ok && lane == 0) {
      // another role gave up: wait (bounded) for the copies in flight before the shared memory goes away
      const uint64_t start = globaltimer();
      for (int s = 0; s < KST; ++s)
        while (issued[s] >= 0 && !mbar_try_wait(smem_u32(&k_full[s]), (uint32_t)issued[s] & 1) &&
               globaltimer() - start < 1000000000ull) {
        }
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issue
    if (elect_one()) {
      constexpr uint32_t idesc_s = mma_idesc(0, C::BM, BN);     // e4m3, K-major A and B
      constexpr uint32_t idesc_o = mma_idesc(0, C::BM, DV, 1);  // f16, A from TMEM, MN-major B (V)
      const uint32_t sq = smem_u32(s_q);
      uint32_t g = 0, nq = 0;  // key tiles and items so far
      for (uint32_t k = 0;; ++k) {
        if (!mbar_wait(&item_full[k & 1], (k >> 1) & 1, a.status)) goto done;
        const int n = works[k & 1].n;
        const bool end = works[k & 1].i < 0;
        mbar_arrive(&item_empty[k & 1]);
        if (end) break;
        if (n == 0) continue;
        if (!mbar_wait(&q_full, nq & 1, a.status)) goto done;
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
              mma_f8_ss(d, kmajor_desc<C::ROW>(sq + half * C::Q_BYTES + c * C::Q_CHUNK + w),
                        kmajor_desc<C::ROW>(sk + c * C::K_CHUNK + w), idesc_s, (half | kk) > 0);
            }
          mma_commit(&k_empty[st]);
          mma_commit(&s_full[G % NS]);
          return true;
        };
        if (!issue_s(0)) goto done;
        for (int j = 0; j < n; ++j) {
          if (j + 1 < n && !issue_s(j + 1)) goto done;
          const uint32_t G = g + j;
          const int st = G % VST;
          if (!mbar_wait(&p_full[G % NS], (G / NS) & 1, a.status)) goto done;
          if (!mbar_wait(&v_full[st], (G / VST) & 1, a.status)) goto done;
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
    }
  } else {
    // ------------------------------------------------------------ conversion of value tiles
    // A warp's pass covers 8 rows x 64 columns: lanes 0-3 the four 16-code pieces of one row, lanes 4-7 of the next,
    // whose f16 pieces fall on the other banks (the swizzle flips with the row's parity).
    constexpr int VP = 8 * C::V_CHUNKS / C::CONV_WARPS;  // passes a warp
    constexpr int AHEAD = 6;                             // tiles between L2 prefetch and use
    const int cw = warp - 6;
    const int sub = lane >> 2, quarter = lane & 3;
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
        const uint8_t* p = v_codes + (int64_t)max(z, 0) * (BN * HD) + w.slice * DV;
#pragma unroll
        for (int s = 0; s < VP; ++s) {
          const int pass = s * C::CONV_WARPS + cw, row = (pass & 7) * 8 + sub, c = pass >> 3;
          vr[s] = z >= 0 && row < keys ? load_codes(p + row * HD + c * 64 + quarter * 16) : make_uint4(0, 0, 0, 0);
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
        uint8_t* tile = s_v + st * C::V_BYTES;
#pragma unroll
        for (int s = 0; s < VP; ++s) {
          const int pass = s * C::CONV_WARPS + cw, row = (pass & 7) * 8 + sub, c = pass >> 3;
          uint8_t* dst = tile + c * C::V_CHUNK + row * 128;
          uint4 lo, hi;
          codes_to_f16(vr[s].x, lo.x, lo.y);
          codes_to_f16(vr[s].y, lo.z, lo.w);
          codes_to_f16(vr[s].z, hi.x, hi.y);
          codes_to_f16(vr[s].w, hi.z, hi.w);
          *reinterpret_cast<uint4*>(dst + (((2 * quarter) ^ (row & 7)) << 4)) = lo;
          *reinterpret_cast<uint4*>(dst + (((2 * quarter + 1) ^ (row & 7)) << 4)) = hi;
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
    // ------------------------------------------------------------ queries, softmax, epilogue (warps 0-3)
    const int r = tid;  // the row within the tile = TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    uint32_t g = 0;
    for (uint32_t k = 0;; ++k) {
      if (!mbar_wait(&item_full[k & 1], (k >> 1) & 1, a.status)) goto done;
      const Work w = works[k & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[k & 1]);
      if (w.i < 0) break;
      const int n = w.n;
      const bool live = r < w.rows, warp_live = warp * 32 < w.rows;
      const int gr = w.r0 + (live ? r : 0);
      const int tok = gr / a.group, head = w.h * a.group + gr - tok * a.group;
      float q_scale = 1.f;
      bool bad = false;  // an infinity or a NaN among the row's queries: NaN wherever it sees a key
      if (n > 0) {
        // The row's queries as hi + lo. The last item's products have read theirs: its last scores were waited for.
        const uint4* src = reinterpret_cast<const uint4*>(a.q + (int64_t)(w.q0 + tok) * a.ldq + (int64_t)head * HD);
        uint32_t top = 0;  // the largest magnitude as a bf16 pattern
        if (live) {
#pragma unroll 4
          for (int c = 0; c < HD / 8; ++c) {
            const uint4 x = src[c];
            const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(v[e] & 0x7fffu, (v[e] >> 16) & 0x7fffu));
          }
        }
        bad = top >= 0x7f80u;
        // the least e with the largest magnitude within 448 = 1.75 * 2^8
        const int e = min(max((int)(top >> 7) - 127 - 8 + ((top & 0x7fu) > 0x60u ? 1 : 0), -120), 120);
        q_scale = pow2i(e);
        const float inv = pow2i(-e);
#pragma unroll 2
        for (int c = 0; c < HD / 16; ++c) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint4 x = live ? src[2 * c + half] : make_uint4(0, 0, 0, 0);
            const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float2 f = unpack_bf16x2(v[2 * y]), h = unpack_bf16x2(v[2 * y + 1]);
              const float4 q4 = make_float4(f.x * inv, f.y * inv, h.x * inv, h.y * inv);
              const uint32_t w0 = e4m3_pair(q4.x, q4.y), w1 = e4m3_pair(q4.z, q4.w);
              hi[2 * half + y] = w0 | (w1 << 16);
              uint32_t h0, h1;
              codes_to_f16(hi[2 * half + y], h0, h1);
              const float2 b0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
              const float2 b1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
              lo[2 * half + y] = e4m3_pair(q4.x - b0.x, q4.y - b0.y) | (e4m3_pair(q4.z - b1.x, q4.w - b1.y) << 16);
            }
          }
          const int at = swizzled<C::ROW>(r, c, C::Q_CHUNK);
          *reinterpret_cast<uint4*>(s_q + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(s_q + C::Q_BYTES + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_async_smem();
        mbar_arrive(&q_full);
      }
      const int off = w.lk - w.lq;
      const int pos0 = w.r0 / a.group + off, pos1 = (w.r0 + w.rows - 1) / a.group + off;  // the tile's first, last row
      const int pos = tok + off;
      const int key_lo = a.left >= 0 ? pos - a.left : 0;
      const int key_hi = a.right >= 0 ? min(w.lk - 1, pos + a.right) : w.lk - 1;
      // running maxima in log2 units, possibly stale by the threshold: of x (the row sum's base) and of x + e_v (O's)
      float m = -INFINITY, big = -INFINITY, l = 0.f;
      Lookup now{-1, 0.f, 0}, ahead{-1, 0.f, 0};
      auto look_up = [&](int j) {
        Lookup x{block_of(a, w, j), 0.f, 0};
        if (x.z >= 0) {
          x.k_scale = a.k_scale[x.z];
          x.v_exp = exponent_of(a.v_scale[x.z]);
        }
        return x;
      };
      if (warp_live) ahead = look_up(lane);
      for (int j = 0; j < n; ++j) {
        if ((j & 31) == 0 && warp_live) {
          now = ahead;
          ahead = look_up(j + 32 + lane);
        }
        const int z = __shfl_sync(0xffffffffu, now.z, j & 31);
        const float ks = __shfl_sync(0xffffffffu, now.k_scale, j & 31);
        const float ve = (float)__shfl_sync(0xffffffffu, now.v_exp, j & 31);
        const uint32_t G = g + j;
        if (!mbar_wait(&s_full[G % NS], (G / NS) & 1, a.status)) goto done;
        if (!warp_live) {  // no row of this warp: its probabilities are never read back
          mbar_arrive(&p_full[G % NS]);
          continue;
        }
        tc_fence_after();
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
        const int key0 = (w.first + j) * BN;
        const bool edge = z < 0 || key0 + BN > w.lk || (a.right >= 0 && key0 + BN - 1 > pos0 + a.right) ||
                          (a.left >= 0 && key0 < pos1 - a.left);
        if (edge) {
          const int lo = z < 0 ? BN : key_lo - key0, hi = key_hi - key0;
#pragma unroll
          for (int e = 0; e < BN; ++e) sv[e] = (e >= lo && e <= hi) ? sv[e] : -INFINITY;
        }
        float mx[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) mx[e] = sv[e];
#pragma unroll
        for (int e = 8; e < BN; e += 2) mx[(e / 2) & 7] = max3(mx[(e / 2) & 7], sv[e], sv[e + 1]);
        const float mraw = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
        const float mul = score_factor(q_scale, ks, a.scale_log2);
        const float mt = mraw == -INFINITY ? -INFINITY : mraw * mul;
        if (mt > m + THRESHOLD) {
          l *= fast_exp2(m - mt);
          m = mt;
        }
        const bool need = mt + ve > big + THRESHOLD;
        const float f = need ? fast_exp2(big - (mt + ve)) : 1.f;
        if (j > 0 && __any_sync(0xffffffffu, need && big != -INFINITY)) {
          if (!mbar_wait(&pv_done[(G - 1) % NS], ((G - 1) / NS) & 1, a.status)) goto done;
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
        const float base = m == -INFINITY ? 0.f : m, vbase = big == -INFINITY ? 0.f : big;
        const float factor = fast_exp2(fminf(base - vbase + ve, 110.f)) * P_SCALE;
        float2 part[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
        const float2 mul2v = make_float2(mul, mul), base2 = make_float2(-base, -base), fac2 = make_float2(factor, factor);
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float2 x = fma2(make_float2(sv[2 * e], sv[2 * e + 1]), mul2v, base2);
          float2 p = make_float2(fast_exp2(x.x), fast_exp2(x.y));
          part[e & 3] = add2(part[e & 3], p);
          p = mul2(p, fac2);
          pk[e] = pack_f16x2(p.x, p.y);
        }
        tmem_st32(s_addr, pk);
        const float2 ps = add2(add2(part[0], part[1]), add2(part[2], part[3]));
        l += ps.x + ps.y;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[G % NS]);
      }
      // ---- epilogue
      if (n > 0) {
        const uint32_t G = g + n - 1;
        if (!mbar_wait(&pv_done[G % NS], (G / NS) & 1, a.status)) goto done;
        tc_fence_after();
      }
      if (warp_live) {
        if (bad && l != 0.f) l = __int_as_float(0x7fffffff);
        const float base = m == -INFINITY ? 0.f : m, vbase = big == -INFINITY ? 0.f : big;
        const int64_t row = w.q0 + tok, col = (int64_t)head * HD + w.slice * DV;
        if (w.slot < 0) {
          const float fin = l == 0.f ? 0.f : fast_exp2(fminf(vbase - base, 126.f)) / (l * P_SCALE);
          const bool gated = a.gate && l != 0.f && live;
          const uint4* gp = reinterpret_cast<const uint4*>(a.gate + row * a.ldg + col);
          uint4* op = reinterpret_cast<uint4*>(a.out + row * a.ldo + col);
#pragma unroll 1
          for (int c = 0; c < DV; c += 32) {
            uint32_t t[32];
            __syncwarp();
            if (n > 0) {
              tmem_ld32(lane_base + C::O_COL + c, t);
              tmem_ld_wait_regs(t);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = l == 0.f ? 0.f : __uint_as_float(t[8 * q + e]) * fin;
              if (gated) {
                const uint4 gv = gp[c / 8 + q];
                const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 s = unpack_bf16x2(gw[e]);
                  x[2 * e] = x_sigmoid(x[2 * e], s.x);
                  x[2 * e + 1] = x_sigmoid(x[2 * e + 1], s.y);
                }
              }
              if (live)
                op[c / 8 + q] = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                           pack_bf16x2(x[6], x[7]));
            }
          }
        } else {
          float* part = a.partials + (int64_t)w.slot * C::PARTIAL;
          if (live) {
            part[C::BM * DV + 3 * r] = m;
            part[C::BM * DV + 3 * r + 1] = big;
            part[C::BM * DV + 3 * r + 2] = l;
          }
#pragma unroll 1
          for (int c = 0; c < DV; c += 32) {
            uint32_t t[32];
            __syncwarp();
            tmem_ld32(lane_base + C::O_COL + c, t);
            tmem_ld_wait_regs(t);
            if (live) {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                *reinterpret_cast<uint4*>(part + r * DV + c + 4 * q) =
                    make_uint4(t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3]);
            }
          }
        }
        // the next item's first product overwrites O: every row of this warp has read it
        tc_fence_before();
      }
      g += n;
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) {
    __syncwarp();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Joins the partials of an item that spans several CTAs' shares. blockIdx.x: the share whose beginning lies inside the
// item, the first such one of the item; blockIdx.y: 32 of its 128 rows, a warp for each fourth. The lanes read the
// partials' statistics together and weigh them; the sums then run in key order with their loads in flight.
template <int HD, int DV>
__global__ void __launch_bounds__(256) join_tiles_kernel(Args a, int ctas) {
  using C = Cfg<HD, DV>;
  constexpr int V = DV / 32;  // columns a lane holds
  const int c = blockIdx.x + 1, lane = threadIdx.x & 31;
  const int64_t total = a.tile_cu[a.n];
  const int np = parts(total, a.group, ctas);
  if (c >= np || total == 0) return;
  const int64_t x = total * c / np;  // share c begins here; share c - 1 ends
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.tile_cu[mid] <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  Item it;
  find<C::SLICES>(a, lo, a.tile_cu[lo], x, it);
  if (it.begin >= x || (c > 1 && total * (c - 1) / np > it.begin)) return;
  const int rows = (int)min((int64_t)128, (int64_t)it.s.lq * a.group - it.tile * 128);
  const Tiles v = visible(a, it.s, it.tile);
  int last = c;  // the last share that meets the item
  {
    // share p holds weight y when floor(p total / np) <= y: the one holding the item's last weight
    last = (int)((it.end * np - 1) / total);
    if (last >= np) last = np - 1;
  }
  const int first = c - 1, n = last - first + 1;
  for (int r = blockIdx.y * 32 + threadIdx.x / 32; r < min(rows, (int)blockIdx.y * 32 + 32); r += 8) {
    const int gr = it.tile * 128 + r;
    const int tok = gr / a.group, head = it.h * a.group + gr - tok * a.group;
    float m = -INFINITY, big = -INFINITY, l = 0.f, o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.f;
    for (int p0 = 0; p0 < n; p0 += 32) {
      const int p = first + p0 + lane;
      float pm = -INFINITY, pb = -INFINITY, pl = 0.f;
      const float* part = a.partials;
      if (p <= last) {
        const int64_t x0 = total * p / np, x1 = total * (p + 1) / np;
        int t0, t1;
        portion(it, max(x0, it.begin), min(x1, it.end), v.n, t0, t1);
        part += (int64_t)(2 * p + (it.begin < x0 ? 0 : 1)) * C::PARTIAL;
        if (t0 < t1) {
          pm = part[C::BM * DV + 3 * r];
          pb = part[C::BM * DV + 3 * r + 1];
          pl = part[C::BM * DV + 3 * r + 2];
        }
      }
      float m_new = pm, big_new = pb;
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) {
        m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, s));
        big_new = fmaxf(big_new, __shfl_xor_sync(0xffffffffu, big_new, s));
      }
      m_new = fmaxf(m_new, m);
      big_new = fmaxf(big_new, big);
      const float base = m_new == -INFINITY ? 0.f : m_new, vbase = big_new == -INFINITY ? 0.f : big_new;
      float sum = pl * fast_exp2(pm - base);
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      l = l * fast_exp2(m - base) + sum;
      const float f0 = fast_exp2(big - vbase), f1 = pb == -INFINITY && pl == 0.f ? -1.f : fast_exp2(pb - vbase);
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] *= f0;
      m = m_new;
      big = big_new;
      const int count = min(32, n - p0);
      const uint64_t mine = reinterpret_cast<uint64_t>(part + r * DV);
#pragma unroll 4
      for (int q = 0; q < count; ++q) {
        const float f = __shfl_sync(0xffffffffu, f1, q);
        const float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, mine, q)) + lane * V;
        if (f < 0.f) continue;  // no key of the row (the partial may hold nothing)
        if constexpr (V >= 4) {
#pragma unroll
          for (int e = 0; e < V; e += 4) {
            const float4 y = *reinterpret_cast<const float4*>(src + e);
            o[e] += y.x * f;
            o[e + 1] += y.y * f;
            o[e + 2] += y.z * f;
            o[e + 3] += y.w * f;
          }
        } else {
          const float2 y = *reinterpret_cast<const float2*>(src);
          o[0] += y.x * f;
          o[1] += y.y * f;
        }
      }
    }
    const float base = m == -INFINITY ? 0.f : m, vbase = big == -INFINITY ? 0.f : big;
    const float fin = l == 0.f ? 0.f : fast_exp2(fminf(vbase - base, 126.f)) / (l * P_SCALE);
    const int64_t row = it.s.q0 + tok, col = (int64_t)head * HD + it.slice * DV + lane * V;
    float y[V];
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = l == 0.f ? 0.f : o[e] * fin;
    if (a.gate && l != 0.f) {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 s = unpack_bf16x2(*reinterpret_cast<const uint32_t*>(a.gate + row * a.ldg + col + e));
        y[e] = x_sigmoid(y[e], s.x);
        y[e + 1] = x_sigmoid(y[e + 1], s.y);
      }
    }
#pragma unroll
    for (int e = 0; e < V; e += 2)
      *reinterpret_cast<uint32_t*>(a.out + row * a.ldo + col + e) = pack_bf16x2(y[e], y[e + 1]);
  }
}

static int64_t header_bytes(int n) { return ((int64_t)(n + 1) * 8 + 15) / 16 * 16; }

template <int HD, int DV>
int64_t workspace(int n, int sms) {
  using C = Cfg<HD, DV>;
  return header_bytes(n) + (int64_t)2 * sms * C::CTAS_PER_SM * C::PARTIAL * (int64_t)sizeof(float);
}

template <int HD, int DV>
int launch(Args a, const void* k_codes, const uint8_t* v_codes, uint8_t* ws, int64_t ws_bytes, cudaStream_t stream) {
  using C = Cfg<HD, DV>;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(KD_ERR_ARGUMENT, "attention_cache: device index");
  const int sms = num_sms(dev), ctas = sms * C::CTAS_PER_SM;
  if (ws_bytes < workspace<HD, DV>(a.n, sms))
    return set_error(KD_ERR_ARGUMENT, "attention_cache: workspace smaller than kd_attention_cache_workspace");
  a.tile_cu = reinterpret_cast<int64_t*>(ws);
  a.partials = reinterpret_cast<float*>(ws + header_bytes(a.n));
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
  join_tiles_kernel<HD, DV><<<dim3(ctas - 1 > 0 ? ctas - 1 : 1, 4), 256, 0, stream>>>(a, ctas);
  return record_cuda_error(cudaGetLastError(), "attention_cache: join launch");
}

}  // namespace ct

namespace ca {

int64_t row_tiles_workspace(int head_dim, int n, int sms) {
  switch (head_dim) {
    case 64: return ct::workspace<64, 64>(n, sms);
    case 128: return ct::workspace<128, 128>(n, sms);
    case 256: return ct::workspace<256, 256>(n, sms);
    default: return ct::workspace<512, 256>(n, sms);
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
