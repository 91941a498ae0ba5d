// Attention of new rows over a cache of e4m3 blocks (cache.cu writes them): for one token of a request up to long
// chunks, GQA, with the end-aligned visibility rule of kd_attention_varlen.
//
// Row i of a request with Lq new rows and Lk cached tokens (the new ones included) sees key j iff
//   i + (Lk - Lq) - left <= j <= i + (Lk - Lq) + right      (left / right < 0: unbounded),
// and with e_k, e_v the exponents of a block's scales
//   x_j = scale * 2^e_k (q . k_j),   o = sum_j exp(x_j - m) 2^e_v v_j / sum_j exp(x_j - m),   m = max_j x_j.
//
// Few query rows per key/value head (the rows of a request that share a head's keys: Lq * Hq / Hkv) are bound by the
// reads of the codes: 2 hd bytes a token and head, once. The work is the list of key tiles (one block of 64 tokens) of
// every (request, key/value head, row tile), in that order; CTA c of P takes the tiles [c, c + 1) * total / P of it, so
// long and short requests balance without the host knowing a length (an item counts ITEM_TILES further tiles, before its
// own, for what it costs beside them). A producer warp reads 32 tiles' table
// entries and scales at a time and keeps a ring of 192 KB filled by TMA; eight warps take the tiles in turn (teams of
// two or four for heads of 256 and 512, each warp a part of the tile's keys), each with a running maximum and sums of
// its own. Each warp leaves a partial result of an item that the CTA goes on from; of the CTA's last item the warps' sums
// become one partial first. A second launch joins them.
//
// The products run on mma.sync.m16n8k16 in f16 with float32 sums, keys and values as the 16-row operand and the query
// rows as the 8 columns: S^T = K Q^T, O^T = V^T P^T. Eight rows then cost half of what a 16-row query tile would, and
// nothing is padded further (a 128-row tcgen05 tile would be mostly empty). The codes turn into f16 exactly, two per
// instruction; ldmatrix hands a thread four neighbouring dims of a key, or two of two keys, and the dims' order within
// the products is permuted to match, so no byte moves but one permute per four value codes. Queries are scaled by a power
// of two per row (exact; f16 holds every bf16 within 2^-24 of the row's largest magnitude). Probabilities are rounded to
// f16 relative to the largest *scaled* probability p 2^e_v met (11 bits, exponents down to 2^-35 of it), so the blocks'
// value scales need no product of their own; the sum of the probabilities stays in float32, unrounded.
#include "cache_attention.cuh"

namespace kd {
namespace ca {

constexpr float THRESHOLD = 4.0f;  // log2 units a row's maximum may grow before its sums are rescaled
constexpr float P_EXPONENT = 11.f, P_SCALE = 2048.f;  // f16 probabilities hold p * 2^11: at most 2^15 with the threshold

constexpr int ITEM_TILES = 8;  // an item's own cost (queries, its partial, the teams' drain) in key tiles: some 6,000 cycles

// HD: head dim. NT: tiles of 8 query rows a warp holds. Registers bound both: a thread holds HD NT / 4 sums of the output
// and the scores of its keys.
template <int HD, int NT>
struct Cfg {
  static constexpr int RT = 8 * NT;                // query rows of an item
  static constexpr int WARPS = 8, THREADS = 32 * (WARPS + 4);  // two warpgroups of consumers, one of producers
  static constexpr int KW = HD <= 64 ? 1 : HD == 128 ? (NT == 1 ? 2 : 1) : HD / 128;  // warps that share a tile by keys
  static constexpr int TEAMS = WARPS / KW;
  static constexpr int MT = BN / KW / 16;          // 16-key tiles of a warp
  static constexpr int BOX = HD < 128 ? HD : 128;  // bytes of a TMA box row (its swizzle span)
  static constexpr int CHUNKS = HD / BOX;
  static constexpr int TILE_BYTES = BN * HD;
  static constexpr int SLOT_BYTES = 2 * TILE_BYTES;
  static constexpr int SLOTS = 192 * 1024 / SLOT_BYTES;
  // A producer takes some 650 cycles a tile, as long as a tile of 16 KB takes to arrive: up to four share the ring. Every
  // slot belongs to one producer, which so sees its uses in order (a parity does not tell laps apart).
  static constexpr int PRODUCERS = HD <= 128 ? 4 : HD == 256 ? 2 : 1;
  static_assert(SLOTS % PRODUCERS == 0, "a slot's uses belong to one producer");
  static_assert(2 * SLOTS % TEAMS == 0, "a team takes every second use of a slot, or every one");
  // Registers: three warpgroups launched at 168; 256 x CONSUMER + 128 x PRODUCER = 384 x 168.
  static constexpr int CONSUMER_REGS = NT * HD >= 512 ? 224 : 208, PRODUCER_REGS = NT * HD >= 512 ? 56 : 88;
  static constexpr int Q_BYTES = RT * HD * 2;      // of one item's queries, in the order of the B fragments
  static constexpr int SMEM = SLOTS * SLOT_BYTES + TEAMS * Q_BYTES + 1024;
  static constexpr int PARTIAL = RT * (HD + 3);    // floats of one warp's partial: O, then (m, M, l) per row
  static_assert(SMEM + 2048 <= 227 * 1024, "shared memory budget");
};

// A request's items: tiles of RT rows of a key/value head, each with the same key tiles.
struct Rows {
  Request r;
  int nrt;
};
template <int RT>
KD_DEVICE Rows rows_of(const Args& a, int i) {
  Rows x;
  x.r = request(a, i);
  x.nrt = (int)(((int64_t)x.r.lq * a.group + RT - 1) / RT);
  return x;
}

// A position in the list of key tiles: request > key/value head > row tile > key tile. `seek(g)` moves forward to the item
// holding tile g.
template <int RT>
struct Cursor {
  int i, h, rt;
  int64_t begin, end;  // the item's tiles
  int item;            // its number over the launch
  Rows x;

  KD_DEVICE void load(const Args& a) {
    while (i < a.n) {
      x = rows_of<RT>(a, i);
      if (x.nrt > 0 && x.r.tiles > 0) break;
      item += x.nrt * a.hkv;
      ++i;
    }
    end = begin + (i < a.n ? x.r.tiles : 0);
  }
  KD_DEVICE void start(const Args& a, int req, int64_t before, int items_before) {
    i = req;
    h = rt = 0;
    begin = before;
    item = items_before;
    load(a);
  }
  KD_DEVICE void seek(const Args& a, int64_t g) {
    if (i < a.n && g >= end && g - end >= x.r.tiles) {  // whole items of this request at once
      const int64_t left = (int64_t)(a.hkv - h) * x.nrt - rt;  // items from this one to the request's last
      const int64_t k = min(left - 1, quotient(g - begin, x.r.tiles));
      const int64_t to = (int64_t)h * x.nrt + rt + k;
      begin += k * x.r.tiles;
      end = begin + x.r.tiles;
      item += (int)k;
      h = (int)quotient(to, x.nrt);
      rt = (int)(to - (int64_t)h * x.nrt);
    }
    while (i < a.n && g >= end) {  // past the request
      begin = end;
      ++item;
      if (++rt == x.nrt) {
        rt = 0;
        if (++h == a.hkv) {
          h = 0;
          ++i;
          load(a);
          if (i < a.n && g >= end) seek_within(a, g);
          continue;
        }
      }
      end = begin + x.r.tiles;
    }
  }
  KD_DEVICE void seek_within(const Args& a, int64_t g) {
    const int64_t k = min((int64_t)a.hkv * x.nrt - 1, quotient(g - begin, x.r.tiles));
    begin += k * x.r.tiles;
    end = begin + x.r.tiles;
    item += (int)k;
    h = (int)quotient(k, x.nrt);
    rt = (int)(k - (int64_t)h * x.nrt);
  }
};

KD_DEVICE void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
KD_DEVICE void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// The transpose of an 8 x 8 matrix of 16-bit elements held two a thread, row by row.
KD_DEVICE uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// d += a (16 x 16, row) * b (16 x 8, column), f16 operands, float32 sums.
KD_DEVICE void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// All consumers.
KD_DEVICE void all_sync(int threads) { asm volatile("bar.sync 9, %0;" ::"r"(threads) : "memory"); }
// The warps of one team.
template <int KW>
KD_DEVICE void team_sync(int team) {
  if constexpr (KW == 1)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * KW) : "memory");
}

// Shared-memory offset of 16-byte piece `c` of row `row` in a tile stored by TMA with BOX-byte rows and BOX-byte
// swizzling, chunk by chunk of BOX bytes.
template <int HD>
KD_DEVICE uint32_t piece(int row, int c) {
  if constexpr (HD == 64) {
    return row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
  } else {
    return (c >> 3) * (BN * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
  }
}

// An item, for the launch that joins its partials.
struct Desc {
  int q0, h, r0, rows;  // the request's first query row, the key/value head, the item's first packed row and their number
  int first, ctas;      // the first CTA's place among the partials, and the CTAs that met the item (0: it has no key tile)
};

// One tile's meta data beside its ring slot.
struct TileInfo {
  float k_scale, v_exp;
  int live;  // 0: the block is absent (a table entry outside the pool): its keys are not seen
  int pad;
};

template <int HD, int NT>
__global__ void __launch_bounds__(Cfg<HD, NT>::THREADS, 1)
    few_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Args a) {
  using C = Cfg<HD, NT>;
  constexpr int SLOTS = C::SLOTS, RT = C::RT, MT = C::MT;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem + SLOTS * C::SLOT_BYTES;  // [TEAMS][Q_BYTES]
  __shared__ uint64_t full[SLOTS], empty[SLOTS];
  __shared__ TileInfo info[SLOTS];
  __shared__ float s_qscale[C::TEAMS][RT];
  __shared__ int64_t s_warp_tiles[C::THREADS / 32], s_before, s_ends[2];
  __shared__ int s_warp_items[C::THREADS / 32], s_req, s_items_before;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  Desc* descs = reinterpret_cast<Desc*>(a.descs);
  if (tid == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], C::KW);
    }
    fence_barrier_init();
  }
  // ---- this CTA's share of the tiles: a scan of the requests' tiles and items for the total, then (a second scan if the
  // requests outnumber the threads) for the share's first request and the tiles at its ends. w counts key tiles of one
  // key/value head; with ITEM_TILES for each item before it, that is the weight that the shares divide.
  int64_t w_mine = 0, w_before = 0, tiles = 0;
  int items_mine = 0, items_before = 0, items = 0;
  auto scan = [&](int i0, int64_t carry, int carry_items) {
    const int i = i0 + tid;
    w_mine = 0;
    items_mine = 0;
    bool falls = false;
    if (i < a.n) {
      falls = a.cu[i + 1] < a.cu[i];
      const Rows r = rows_of<RT>(a, i);
      w_mine = (int64_t)r.nrt * r.r.tiles;
      items_mine = r.nrt;
    }
    int64_t x = w_mine;
    int y = items_mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t px = __shfl_up_sync(0xffffffffu, x, o);
      const int py = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += px;
        y += py;
      }
    }
    if (lane == 31) {
      s_warp_tiles[warp] = x;
      s_warp_items[warp] = y;
    }
    falls = __syncthreads_or(falls) || carry < 0;
    w_before = carry + x - w_mine;
    items_before = carry_items + y - items_mine;
#pragma unroll
    for (int v = 0; v < C::THREADS / 32; ++v) {
      if (v < warp) {
        w_before += s_warp_tiles[v];
        items_before += s_warp_items[v];
      }
      carry += s_warp_tiles[v];
      carry_items += s_warp_items[v];
    }
    __syncthreads();
    tiles = falls ? -1 : carry;
    items = carry_items;
  };
  for (int i0 = 0; i0 < a.n; i0 += C::THREADS) scan(i0, tiles, items);
  // Bounds that fall name rows twice: more items than the workspace holds. Such a launch has no work.
  if (tiles < 0) {
    if (tid == 0 && blockIdx.x == 0) *a.items = 0;
    return;
  }
  const int64_t total = (tiles + (int64_t)ITEM_TILES * items) * a.hkv;
  const int np = (int)shares(total, gridDim.x);
  const int64_t v_lo = quotient(total * blockIdx.x, np);
  const int64_t v_hi = (int)blockIdx.x < np ? quotient(total * (blockIdx.x + 1), np) : v_lo;
  if (tid == 0) s_ends[0] = s_ends[1] = tiles * a.hkv;  // a bound past the last request
  __syncthreads();
  if (a.n > C::THREADS) tiles = items = 0;
  for (int i0 = 0; i0 < a.n; i0 += C::THREADS) {
    if (a.n > C::THREADS) scan(i0, tiles, items);
    const int i = i0 + tid;
    if (items_mine > 0) {
      if (w_mine == 0 && blockIdx.x == 0) {  // rows that see no key: for the launch that joins the partials
        const Rows x = rows_of<RT>(a, i);
        for (int k = 0; k < items_mine * a.hkv; ++k) {
          const int h = k / items_mine, r0 = (k - h * items_mine) * RT;
          descs[items_before * a.hkv + k] = Desc{x.r.q0, h, r0, min(RT, x.r.lq * a.group - r0), 0, 0};
        }
      }
      const int64_t v = (w_before + (int64_t)ITEM_TILES * items_before) * a.hkv;  // the request's weights
      const int64_t own = w_mine + (int64_t)ITEM_TILES * items_mine;
      const int64_t per = own / items_mine, mine = w_mine / items_mine;            // an item's weight, its tiles
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t x = (e ? v_hi : v_lo) - v;
        if (x >= 0 && x < own * a.hkv) {
          const int64_t k = quotient(x, per);
          s_ends[e] = w_before * a.hkv + k * mine + max((int64_t)0, x - k * per - ITEM_TILES);
          if (e == 0) {
            s_req = i;
            s_before = w_before * a.hkv;
            s_items_before = items_before * a.hkv;
          }
        }
      }
    }
  }
  if (tid == 0 && blockIdx.x == 0) *a.items = items * a.hkv;
  __syncthreads();
  const int64_t lo = s_ends[0], hi = s_ends[1];
  if (lo >= hi) return;

  Cursor<RT> c;
  if (warp >= C::WARPS) {
    set_registers_down<C::PRODUCER_REGS>();
    const int me = warp - C::WARPS;
    if (me >= C::PRODUCERS) return;
    c.start(a, s_req, s_before, s_items_before);
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
    }
    // This producer's k-th tile is lo + k PRODUCERS + me; each lane looks up one tile's block and scales, 32 ahead.
    const uint32_t mine = hi - lo > me ? (uint32_t)((hi - lo - me + C::PRODUCERS - 1) / C::PRODUCERS) : 0;
    uint32_t issued = mine;
    int z = -1, next_z = -1, ve = 0, next_ve = 0;
    float ks = 0.f, next_ks = 0.f;
    auto look_up = [&](uint32_t k) {
      next_z = -1;
      next_ks = 0.f;
      next_ve = 0;
      if (k < mine) {
        const int64_t g = lo + (int64_t)k * C::PRODUCERS + me;
        c.seek(a, g);
        const int id = a.table[(int64_t)c.i * a.ldt + c.x.r.first + (int)(g - c.begin)];
        if (id >= 0 && id < a.blocks) {
          next_z = id * a.hkv + c.h;
          next_ks = a.k_scale[next_z];
          next_ve = exponent_of(a.v_scale[next_z]);
        }
      }
    };
    look_up(lane);
    for (uint32_t k0 = 0; k0 < mine; k0 += 32) {
      z = next_z;
      ks = next_ks;
      ve = next_ve;
      look_up(k0 + 32 + lane);
      const uint32_t some = min(32u, mine - k0);
      for (uint32_t j = 0; j < some; ++j) {
        const uint32_t at = (k0 + j) * C::PRODUCERS + me, slot = at % SLOTS;
        const int zz = __shfl_sync(0xffffffffu, z, j);
        const float s = __shfl_sync(0xffffffffu, ks, j);
        const int e = __shfl_sync(0xffffffffu, ve, j);
        bool ok = true;
        if (lane == 0) {
          ok = mbar_wait(&empty[slot], ((at / SLOTS) & 1) ^ 1, a.status);
          if (ok) {
            info[slot] = TileInfo{s, (float)e, zz >= 0, 0};
            if (zz >= 0) {
              mbar_arrive_expect_tx(&full[slot], C::SLOT_BYTES);
              uint8_t* dst = smem + slot * C::SLOT_BYTES;
              for (int x = 0; x < C::CHUNKS; ++x) {
                tma_load_3d(&map_k, &full[slot], dst + x * BN * C::BOX, x * C::BOX, 0, zz);
                tma_load_3d(&map_v, &full[slot], dst + C::TILE_BYTES + x * BN * C::BOX, x * C::BOX, 0, zz);
              }
            } else {
              mbar_arrive(&full[slot]);
            }
          }
        }
        if (!__shfl_sync(0xffffffffu, ok, 0)) {
          issued = k0 + j;  // a consumer gave up
          goto drain;
        }
      }
    }
  drain:
    // Wait (bounded) for this producer's copies in flight, the last one into each of its slots: consumers that gave up do
    // not wait for them before the shared memory goes away.
    if (lane == 0) {
      const uint64_t start = globaltimer();
      for (uint32_t k = issued > SLOTS / C::PRODUCERS ? issued - SLOTS / C::PRODUCERS : 0; k < issued; ++k) {
        const uint32_t at = k * C::PRODUCERS + me;
        while (!mbar_try_wait(smem_u32(&full[at % SLOTS]), (at / SLOTS) & 1) && globaltimer() - start < 1000000000ull) {
        }
      }
    }
    return;
  }

  // ------------------------------------------------------------ consumers
  set_registers_up<C::CONSUMER_REGS>();
  c.start(a, s_req, s_before, s_items_before);
  const int team = warp / C::KW, part_of = warp % C::KW;
  const int row_g = lane >> 2, t4 = lane & 3;  // fragments: row_g a key or dim (and key + 8), 2 t4 and 2 t4 + 1 query rows
  const uint32_t ring = smem_u32(smem);
  c.seek(a, lo);
  uint32_t at = team;  // the team's next tile, counted from the CTA's first
  bool dead = false;   // a wait gave up: walk on to the end without computing, so that no warp waits at a barrier alone
  uint2* qf = reinterpret_cast<uint2*>(s_q + team * C::Q_BYTES);
  // Teams walk the items on their own: one that is done with an item goes on to the next while others finish.
  for (int64_t g = lo; g < hi;) {
    const int64_t stop = min(c.end, hi);  // the fragment of this item: tiles [g, stop)
    const int lq = c.x.r.lq, lk = c.x.r.lk;
    const int rows = min(RT, lq * a.group - c.rt * RT);
    if (g == c.begin && tid == 0) {
      // the weight at the item's first tile is c.begin + ITEM_TILES * (its number + 1); the last tile's CTA as in the shares
      const int64_t v = c.begin + (int64_t)ITEM_TILES * (c.item + 1) + c.x.r.tiles;
      const int last = (int)quotient(v * np - 1, total);
      descs[c.item] = Desc{c.x.r.q0, c.h, c.rt * RT, rows, c.item + (int)blockIdx.x, last - (int)blockIdx.x + 1};
    }
    if ((int64_t)at + lo < stop) {
      // ---- queries: f16, scaled to the row's largest magnitude, in the order of the B fragments; RT / KW rows a warp, LPR
      // lanes a row, each every LPR-th piece of 8 dims
      constexpr int MINE = RT / C::KW, LPR = MINE >= 32 ? 1 : 32 / MINE, PIECES = HD / 8 / LPR > 0 ? HD / 8 / LPR : 1;
      static_assert(MINE <= 32, "a lane has one row");
      team_sync<C::KW>(team);  // the team has left its last item, whose queries these replace
      const int rr = part_of * MINE + lane / LPR, first = lane % LPR, r = c.rt * RT + rr;
      const int tok = r / a.group;
      const __nv_bfloat16* src = a.q + (int64_t)(c.x.r.q0 + tok) * a.ldq + (int64_t)(c.h * a.group + r - tok * a.group) * HD;
      uint4 w[PIECES];
      uint32_t top = 0;  // the largest magnitude as a bf16 pattern
#pragma unroll
      for (int u = 0; u < PIECES; ++u) {
        const int d8 = u * LPR + first;
        w[u] = rr < rows && d8 < HD / 8 ? reinterpret_cast<const uint4*>(src)[d8] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < PIECES; ++u) {
        const uint32_t x[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(x[e] & 0x7fffu, (x[e] >> 16) & 0x7fffu));
      }
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int e = max((int)(top >> 7) - 127, -120);
      // An infinity or a NaN makes every element NaN, so that the row is NaN wherever it sees a key: an infinity's own
      // scores may all be -inf, which would read as nothing seen.
      const float inv = top >= 0x7f80u ? __int_as_float(0x7fffffff) : pow2i(-e);
      if (first == 0) s_qscale[team][rr] = pow2i(e) * a.scale_log2;
#pragma unroll
      for (int u = 0; u < PIECES; ++u) {
        const int d8 = u * LPR + first;  // dims 8 d8 ..: step d8 / 2, threads 2 (d8 % 2) and the next of the fragment
        if (d8 < HD / 8) {
          const float2 p0 = unpack_bf16x2(w[u].x), p1 = unpack_bf16x2(w[u].y), p2 = unpack_bf16x2(w[u].z),
                       p3 = unpack_bf16x2(w[u].w);
          *reinterpret_cast<uint4*>(qf + ((d8 >> 1) * NT + (rr >> 3)) * 32 + (rr & 7) * 4 + (d8 & 1) * 2) =
              make_uint4(pack_f16x2(p0.x * inv, p0.y * inv), pack_f16x2(p1.x * inv, p1.y * inv),
                         pack_f16x2(p2.x * inv, p2.y * inv), pack_f16x2(p3.x * inv, p3.y * inv));
        }
      }
      team_sync<C::KW>(team);
    }
    // the item's rows from the first to the last: which key tiles need a mask
    const int pos0 = c.rt * RT / a.group + lk - lq;
    const int pos1 = (c.rt * RT + rows - 1) / a.group + lk - lq;

    float m[NT][2], big[NT][2], l[NT][2];  // running maxima (log2 units, possibly stale) of x and of x + e_v; row sums
    float o[HD / 16][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = big[nt][0] = big[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int x = 0; x < HD / 16; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x][nt][e] = 0.f;
    }
    bool met = false;
    for (; (int64_t)at + lo < stop; at += C::TEAMS) {
      const uint32_t slot = at % SLOTS;
      // A team may be a lap ahead of the team that takes the slot's tile before this one, and a parity cannot tell the
      // phase before from the one after: that tile's release first, then this one's arrival.
      const uint32_t lap = at / SLOTS;
      dead = dead || (lap > 0 && !mbar_wait(&empty[slot], (lap - 1) & 1, a.status)) ||
             !mbar_wait(&full[slot], lap & 1, a.status);
      if (__any_sync(0xffffffffu, dead)) {
        dead = true;
        continue;
      }
      const TileInfo ti = info[slot];
      const uint32_t sk = ring + slot * C::SLOT_BYTES, sv = sk + C::TILE_BYTES;
      const int tile0 = (c.x.r.first + (int)((int64_t)at + lo - c.begin)) * BN;
      const int key_off = part_of * (16 * MT), key0 = tile0 + key_off;  // the warp's first key in the tile, in the request
      if (ti.live && key0 < lk) {
        met = true;
        // ---- S^T = K Q^T: 16 keys a tile; a thread holds keys row_g and row_g + 8 of its rows 2 t4 and 2 t4 + 1
        float s[MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
        auto keys = [&](int mt, uint32_t w0, uint32_t w1, const uint2 (&q2)[NT]) {
          uint32_t af[4];
          codes_to_f16(w0, af[0], af[2]);
          codes_to_f16(w1, af[1], af[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(s[mt][nt], af, q2[nt].x, q2[nt].y);
        };
        if constexpr (MT >= 2) {
#pragma unroll 8
          for (int x = 0; x < HD / 16; ++x) {
            uint2 q2[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) q2[nt] = qf[(x * NT + nt) * 32 + lane];
#pragma unroll
            for (int mt = 0; mt < MT; mt += 2) {
              uint32_t w[4];
              ldmatrix4(sk + piece<HD>(key_off + mt * 16 + lane, x), w);
              keys(mt, w[0], w[1], q2);
              keys(mt + 1, w[2], w[3], q2);
            }
          }
        } else {
#pragma unroll 8
          for (int x = 0; x < HD / 16; x += 2) {
            uint32_t w[4];
            ldmatrix4(sk + piece<HD>(key_off + (lane & 15), x + (lane >> 4)), w);
            uint2 q2[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) q2[nt] = qf[(x * NT + nt) * 32 + lane];
            keys(0, w[0], w[1], q2);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) q2[nt] = qf[((x + 1) * NT + nt) * 32 + lane];
            keys(0, w[2], w[3], q2);
          }
        }
        const bool tail = key0 + 16 * MT > lk;  // places past the request's tokens hold anything
        const bool edge = tail || (a.right >= 0 && key0 + 16 * MT - 1 > pos0 + a.right) ||
                          (a.left >= 0 && key0 < pos1 - a.left);
        // ---- softmax
        float mt_new[NT][2];
        bool need = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int rr = nt * 8 + 2 * t4 + u;
            const float mul = score_factor(s_qscale[team][rr], ti.k_scale);
            int key_lo = 0, key_hi = 0;
            if (edge) {
              const int pos = (c.rt * RT + rr) / a.group + lk - lq;
              key_lo = a.left >= 0 ? pos - a.left : 0;
              key_hi = a.right >= 0 ? min(lk - 1, pos + a.right) : lk - 1;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float x = s[mt][nt][2 * e + u] * mul;
                if (edge) {
                  const int key = key0 + mt * 16 + 8 * e + row_g;
                  x = key >= key_lo && key <= key_hi ? x : -INFINITY;
                }
                s[mt][nt][2 * e + u] = x;
                mx = fmaxf(mx, x);
              }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mt_new[nt][u] = mx;
            need |= mx + ti.v_exp > big[nt][u] + THRESHOLD || mx > m[nt][u] + THRESHOLD;
          }
        if (__any_sync(0xffffffffu, need)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float alpha[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float mx = mt_new[nt][u], mv = mx + ti.v_exp;
              if (mx > m[nt][u] + THRESHOLD) {
                l[nt][u] *= fast_exp2(m[nt][u] - mx);
                m[nt][u] = mx;
              }
              alpha[u] = 1.f;
              if (mv > big[nt][u] + THRESHOLD) {
                alpha[u] = fast_exp2(big[nt][u] - mv);
                big[nt][u] = mv;
              }
            }
#pragma unroll
            for (int x = 0; x < HD / 16; ++x) {
              o[x][nt][0] *= alpha[0];
              o[x][nt][1] *= alpha[1];
              o[x][nt][2] *= alpha[0];
              o[x][nt][3] *= alpha[1];
            }
          }
        }
        uint32_t pb[MT][NT][2];  // P^T as B fragments
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float base[2], factor[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            base[u] = m[nt][u] == -INFINITY ? 0.f : m[nt][u];
            const float vbase = big[nt][u] == -INFINITY ? 0.f : big[nt][u];
            factor[u] = fast_exp2(fminf(base[u] - vbase + ti.v_exp + P_EXPONENT, 126.f));
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              p[e] = fast_exp2(s[mt][nt][e] - base[e & 1]);
              l[nt][e & 1] += p[e];
              p[e] *= factor[e & 1];
            }
            pb[mt][nt][0] = transpose8(pack_f16x2(p[0], p[1]));
            pb[mt][nt][1] = transpose8(pack_f16x2(p[2], p[3]));
          }
        }
        // ---- O^T += V^T P^T: 16 keys a step; a 16-dim piece gives the even dims (rows 0-7) and the odd ones (8-15)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          // codes of places past the request's last token are cleared: a probability of 0 times a NaN code is NaN
          uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
          if (tail) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int left_keys = lk - (key0 + mt * 16 + y * 8 + 2 * t4);
              keep[y] = left_keys >= 2 ? 0xffffffffu : left_keys == 1 ? 0x0000ffffu : 0u;
            }
          }
#pragma unroll
          for (int x = 0; x < HD / 16; x += 2) {
            uint32_t w[4];  // (keys 0-7, keys 8-15) of piece x, then of x + 1
            ldmatrix4_trans(sv + piece<HD>(key_off + mt * 16 + (lane & 15), x + (lane >> 4)), w);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t af[4];
              codes_to_f16(__byte_perm(w[2 * y] & keep[0], 0, 0x3120), af[0], af[1]);
              codes_to_f16(__byte_perm(w[2 * y + 1] & keep[1], 0, 0x3120), af[2], af[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16(o[x + y][nt], af, pb[mt][nt][0], pb[mt][nt][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot]);
    }
    // ---- the partials of this fragment: item + CTA number their place (both only grow along the list)
    float* place = a.partials + (int64_t)(c.item + (int)blockIdx.x) * C::WARPS * C::PARTIAL;
    float sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x = l[nt][u];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        sum[nt][u] = x + __shfl_xor_sync(0xffffffffu, x, 16);
      }
    if (stop < hi) {
      // more items follow: each warp leaves its own and goes on
      float* part = place + warp * C::PARTIAL;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int rr = nt * 8 + 2 * t4 + u;
          if (rr < rows) {
            if (row_g == 0) {
              float* st = part + RT * HD + 3 * rr;
              st[0] = m[nt][u];
              st[1] = big[nt][u];
              st[2] = sum[nt][u];
            }
            if (met) {
#pragma unroll
              for (int x = 0; x < HD / 16; ++x)
                *reinterpret_cast<float2*>(part + rr * HD + 16 * x + 2 * row_g) = make_float2(o[x][nt][u], o[x][nt][2 + u]);
            }
          }
        }
    } else {
      // the CTA's last: the warps' sums become one partial, in the ring, which every tile has left
      constexpr int LD = HD + 8;  // floats between rows
      static_assert(C::WARPS * RT * (LD + 3) * 4 <= SLOTS * C::SLOT_BYTES, "the ring holds the warps' sums");
      float* all = reinterpret_cast<float*>(smem);
      float* stats = all + C::WARPS * RT * LD;  // [3][WARPS][RT]
      all_sync(32 * C::WARPS);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int rr = nt * 8 + 2 * t4 + u;
          if (row_g == 0) {
            stats[warp * RT + rr] = m[nt][u];
            stats[(C::WARPS + warp) * RT + rr] = big[nt][u];
            stats[(2 * C::WARPS + warp) * RT + rr] = sum[nt][u];
          }
#pragma unroll
          for (int x = 0; x < HD / 16; ++x)
            *reinterpret_cast<float2*>(all + (warp * RT + rr) * LD + 16 * x + 2 * row_g) =
                make_float2(o[x][nt][u], o[x][nt][2 + u]);
        }
      all_sync(32 * C::WARPS);
      for (int i = tid; i < rows * (HD / 4); i += 32 * C::WARPS) {
        const int rr = i / (HD / 4), d = (i - rr * (HD / 4)) * 4;
        float mm = -INFINITY, bb = -INFINITY;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) {
          mm = fmaxf(mm, stats[w * RT + rr]);
          bb = fmaxf(bb, stats[(C::WARPS + w) * RT + rr]);
        }
        const float base = mm == -INFINITY ? 0.f : mm, vbase = bb == -INFINITY ? 0.f : bb;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float ll = 0.f;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) {
          ll += stats[(2 * C::WARPS + w) * RT + rr] * fast_exp2(stats[w * RT + rr] - base);
          const float f = fast_exp2(stats[(C::WARPS + w) * RT + rr] - vbase);
          const float4 y = *reinterpret_cast<const float4*>(all + (w * RT + rr) * LD + d);
          acc.x += y.x * f;
          acc.y += y.y * f;
          acc.z += y.z * f;
          acc.w += y.w * f;
        }
        *reinterpret_cast<float4*>(place + rr * HD + d) = acc;
        if (d < 32) {  // the row's statistics, and the other warps' places marked empty, by eight threads
          const int w = d / 4;
          float* st = place + w * C::PARTIAL + RT * HD + 3 * rr;
          st[0] = w ? -INFINITY : mm;
          st[1] = w ? -INFINITY : bb;
          st[2] = w ? 0.f : ll;
        }
      }
    }
    g = stop;
    c.seek(a, g);
  }
}

// Joins an item's partials. A warp has 128 columns (64 for heads of 64) of a row, so a block RB rows; where the item has
// fewer, several warps share a row and each takes every WPR-th partial. The lanes read all the partials' statistics of the
// row together, then four columns each of the partials, in key order, eight loads in flight.
template <int HD, int NT>
__global__ void __launch_bounds__(256) join_kernel(Args a) {
  using C = Cfg<HD, NT>;
  constexpr int RT = C::RT, CW = HD <= 128 ? 1 : HD / 128, RB = 8 / CW, V = HD == 64 ? 2 : 4;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the partials are there after this
  const int items = *a.items;
  const Desc d = reinterpret_cast<const Desc*>(a.descs)[blockIdx.x];
  const int r0 = blockIdx.y * RB;
  if ((int)blockIdx.x >= items || r0 >= d.rows) return;
  // Every CTA but the last left one partial (it went on to no other item), the last one eight, if only one that counts.
  const int n = d.ctas ? d.ctas - 1 + C::WARPS : 0;
  auto place = [&](int q) -> const float* {
    const int c = min(q, d.ctas - 1);
    return a.partials + ((int64_t)(d.first + c) * C::WARPS + (q - c)) * C::PARTIAL;
  };
  const int here = min(RB, d.rows - r0);
  const int wpr = here * 2 > RB ? 1 : here * 4 > RB ? 2 : here * 8 > RB ? 4 : 8;  // warps of a row's columns
  const int unit = warp / CW, col = (warp % CW) * 128 + lane * V;
  const int sub = unit % wpr, row = r0 + unit / wpr;
  const bool live = row < d.rows;
  const int gr = d.r0 + (live ? row : 0), tok = gr / a.group, head = d.h * a.group + gr - tok * a.group;
  uint2 gate = make_uint2(0, 0);
  if (a.gate && live) {
    const __nv_bfloat16* src = a.gate + (int64_t)(d.q0 + tok) * a.ldg + (int64_t)head * HD + col;
    if constexpr (V == 4)
      gate = *reinterpret_cast<const uint2*>(src);
    else
      gate.x = *reinterpret_cast<const uint32_t*>(src);
  }
  float acc[V], l = 0.f, m = -INFINITY, big = -INFINITY;
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  if (live) {
    for (int q0 = lane; q0 < n; q0 += 128) {  // four loads in flight
      float x[4], y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* st = place(min(q0 + 32 * u, n - 1)) + RT * HD + 3 * row;
        x[u] = q0 + 32 * u < n ? st[0] : -INFINITY;
        y[u] = q0 + 32 * u < n ? st[1] : -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        m = fmaxf(m, x[u]);
        big = fmaxf(big, y[u]);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
    }
    const float base = m == -INFINITY ? 0.f : m, vbase = big == -INFINITY ? 0.f : big;
    for (int q0 = lane; q0 < n; q0 += 128) {
      float x[4], y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* st = place(min(q0 + 32 * u, n - 1)) + RT * HD + 3 * row;
        x[u] = q0 + 32 * u < n ? st[0] : -INFINITY;
        y[u] = q0 + 32 * u < n ? st[2] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) l += y[u] * fast_exp2(x[u] - base);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const int mine = n > sub ? (n - sub + wpr - 1) / wpr : 0;  // this warp's partials: sub, sub + wpr, ..
    for (int k0 = 0; k0 < mine; k0 += 32) {
      float f = -1.f;  // < 0: the warp that left it met no key of the row (its sums may hold anything)
      if (k0 + lane < mine) {
        const float* st = place(sub + (k0 + lane) * wpr) + RT * HD + 3 * row;
        if (st[1] != -INFINITY || st[2] != 0.f) f = fast_exp2(st[1] - vbase);
      }
      const int some = min(32, mine - k0);
      for (int k1 = 0; k1 < some; k1 += 8) {
        float4 y[8];
        float w[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          w[q] = __shfl_sync(0xffffffffu, f, (k1 + q) & 31);
          if (k1 + q >= some) w[q] = -1.f;
          y[q] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (!(w[q] < 0.f)) {
            const float* src = place(sub + (k0 + k1 + q) * wpr) + row * HD + col;
            if constexpr (V == 4) {
              y[q] = *reinterpret_cast<const float4*>(src);
            } else {
              const float2 t = *reinterpret_cast<const float2*>(src);
              y[q].x = t.x;
              y[q].y = t.y;
            }
          }
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float x = w[q] < 0.f ? 0.f : w[q];
          acc[0] += y[q].x * x;
          acc[1] += y[q].y * x;
          if constexpr (V == 4) {
            acc[2] += y[q].z * x;
            acc[3] += y[q].w * x;
          }
        }
      }
    }
  }
  if (wpr > 1) {
    __shared__ float s_o[8][V][32];
#pragma unroll
    for (int e = 0; e < V; ++e) s_o[warp][e][lane] = acc[e];
    __syncthreads();
    if (sub > 0) return;
    for (int w = 1; w < wpr; ++w)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += s_o[warp + w * CW][e][lane];
  }
  if (!live) return;
  // o = O 2^(M - m) / (2^11 l); without a visible key 0
  const float base = m == -INFINITY ? 0.f : m, vbase = big == -INFINITY ? 0.f : big;
  const float fin = l == 0.f ? 0.f : fast_exp2(fminf(vbase - base, 126.f)) / (l * P_SCALE);
  uint32_t out[V / 2];
#pragma unroll
  for (int y = 0; y < V / 2; ++y) {
    float2 v = l == 0.f ? make_float2(0.f, 0.f) : make_float2(acc[2 * y] * fin, acc[2 * y + 1] * fin);
    if (a.gate && l != 0.f) {
      const float2 s = unpack_bf16x2(y ? gate.y : gate.x);
      v.x = x_sigmoid(v.x, s.x);
      v.y = x_sigmoid(v.y, s.y);
    }
    out[y] = pack_bf16x2(v.x, v.y);
  }
  __nv_bfloat16* dst = a.out + (int64_t)(d.q0 + tok) * a.ldo + (int64_t)head * HD + col;
  if constexpr (V == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(out[0], out[1]);
  else
    *reinterpret_cast<uint32_t*>(dst) = out[0];
}

// The 8-row tiles of this file's kernel for these requests, 0 for the kernel with 128-row tiles; both are right for any
// rows. Measured (us, this file's / the other, 8 requests of 16,384 tokens, 8 key/value heads): head 64, 16 rows 54 / 63,
// 24 rows 96 / 64; head 128, 16 rows 66 / 79; head 256, 16 rows 113 / 141. Heads of 512 hold 8 rows; 16 rows read the
// codes twice, the second time from L2.
static int row_tiles_of_8(int max_q, int group, int head_dim) {
  const int64_t rows = (int64_t)max_q * group;
  return rows > 16 ? 0 : rows <= 8 || head_dim == 512 ? 1 : 2;
}

// Bytes of scratch: the number of items, their descriptions, the warps' partials per (item + CTA).
static int64_t header_bytes(int64_t items) { return 16 + (items * (int64_t)sizeof(Desc) + 15) / 16 * 16; }

template <int HD, int NT>
int64_t items_bound(int n, int64_t total_q, int hkv, int group) {
  return (total_q * group / Cfg<HD, NT>::RT + n) * hkv;
}
template <int HD, int NT>
int64_t workspace_bytes(int n, int64_t total_q, int hkv, int group, int ctas) {
  using C = Cfg<HD, NT>;
  const int64_t items = items_bound<HD, NT>(n, total_q, hkv, group);
  return header_bytes(items) + (items + ctas) * C::WARPS * C::PARTIAL * (int64_t)sizeof(float);
}

template <int HD, int NT>
int launch(Args a, const void* k_codes, const void* v_codes, uint8_t* ws, int64_t ws_bytes, cudaStream_t stream) {
  using C = Cfg<HD, NT>;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(KD_ERR_ARGUMENT, "attention_cache: device index");
  const int ctas = num_sms(dev);
  const int64_t items = items_bound<HD, NT>(a.n, a.total_q, a.hkv, a.group);
  if ((items + ctas) * C::WARPS > 0x7fffffff) return set_error(KD_ERR_ARGUMENT, "attention_cache: too many row tiles");
  if (ws_bytes < workspace_bytes<HD, NT>(a.n, a.total_q, a.hkv, a.group, ctas))
    return set_error(KD_ERR_ARGUMENT, "attention_cache: workspace smaller than kd_attention_cache_workspace");
  a.items = reinterpret_cast<int*>(ws);
  a.descs = ws + 16;
  a.partials = reinterpret_cast<float*>(ws + header_bytes(items));
  CUtensorMap mk, mv;
  const auto dt = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const auto sw = HD == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  int rc = make_tma_3d(&mk, k_codes, dt, 1, HD, BN, (uint64_t)a.blocks * a.hkv, HD, (uint64_t)BN * HD, C::BOX, BN, 1,
                       sw);
  if (!rc)
    rc = make_tma_3d(&mv, v_codes, dt, 1, HD, BN, (uint64_t)a.blocks * a.hkv, HD, (uint64_t)BN * HD, C::BOX, BN, 1, sw);
  if (rc) return rc;
  auto kernel = few_rows_kernel<HD, NT>;
  static bool configured[64] = {false};
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return record_cuda_error(e, "attention_cache: cudaFuncSetAttribute");
    configured[dev] = true;
  }
  kernel<<<ctas, C::THREADS, C::SMEM, stream>>>(mk, mv, a);
  rc = record_cuda_error(cudaGetLastError(), "attention_cache: launch");
  if (rc) return rc;
  return launch_after(join_kernel<HD, NT>, dim3((unsigned)items, C::RT * HD / (HD <= 128 ? 8 * HD : 1024)), 256, stream,
                      a);
}

// f(head dim, 8-row tiles) with both as constants.
template <typename F>
auto with_kernel(int head_dim, int nt, F f) {
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  switch (head_dim) {
    case 64: return nt == 1 ? f(std::integral_constant<int, 64>{}, one) : f(std::integral_constant<int, 64>{}, two);
    case 128: return nt == 1 ? f(std::integral_constant<int, 128>{}, one) : f(std::integral_constant<int, 128>{}, two);
    case 256: return nt == 1 ? f(std::integral_constant<int, 256>{}, one) : f(std::integral_constant<int, 256>{}, two);
    default: return f(std::integral_constant<int, 512>{}, one);
  }
}

}  // namespace ca
}  // namespace kd

using namespace kd;

extern "C" int kd_attention_cache_workspace(int num_requests, int max_q, int64_t total_q, int num_heads_q,
                                            int num_heads_kv, int head_dim, int64_t* bytes) {
  if (!bytes || num_requests < 0 || max_q < 0 || total_q < 0 || num_heads_q <= 0 || num_heads_kv <= 0 ||
      num_heads_q % num_heads_kv)
    return set_error(KD_ERR_ARGUMENT, "attention_cache_workspace: sizes, heads or a null pointer");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512)
    return set_error(KD_ERR_ARGUMENT, "attention_cache_workspace: head_dim must be 64, 128, 256 or 512");
  int dev = 0;
  if (int rc = record_cuda_error(cudaGetDevice(&dev), "attention_cache_workspace: device")) return rc;
  const int sms = num_sms(dev), group = num_heads_q / num_heads_kv;
  const int nt = ca::row_tiles_of_8(max_q, group, head_dim);
  *bytes = nt == 0 ? ca::row_tiles_workspace(head_dim, sms)
                   : ca::with_kernel(head_dim, nt, [&](auto hd, auto t) {
                       return ca::workspace_bytes<hd(), t()>(num_requests, total_q, num_heads_kv, group, sms);
                     });
  return KD_OK;
}

extern "C" int kd_attention_cache(const void* q, int64_t ldq, const void* k_codes, const void* v_codes,
                                  const float* k_scale, const float* v_scale, int64_t num_blocks, const int32_t* table,
                                  int64_t ld_table, int table_width, const int32_t* cu_q, const int32_t* kv_len,
                                  int num_requests, int max_q, int64_t total_q, void* out, int64_t ldo,
                                  const void* gate, int64_t ldg, int num_heads_q, int num_heads_kv, int head_dim,
                                  float scale, int window_left, int window_right, void* workspace,
                                  int64_t workspace_bytes, int* status, cudaStream_t stream) {
  if (num_requests < 0 || max_q < 0 || total_q < 0 || total_q > 0x3fffffff || num_blocks < 0 || table_width < 0 ||
      ld_table < table_width)
    return set_error(KD_ERR_ARGUMENT, "attention_cache: negative sizes, or a table narrower than its width");
  if (num_requests == 0 || total_q == 0) return KD_OK;
  if (num_heads_q <= 0 || num_heads_kv <= 0 || num_heads_q % num_heads_kv)
    return set_error(KD_ERR_ARGUMENT, "attention_cache: query heads must be a multiple of key/value heads");
  if (num_blocks == 0 || num_blocks * num_heads_kv > 0x7fffffff || (int64_t)table_width * KD_KV_BLOCK > 0x3fffffff)
    return set_error(KD_ERR_ARGUMENT, "attention_cache: 1 to 2^31 - 1 blocks x heads, below 2^30 tokens in a table row");
  if (!q || !k_codes || !v_codes || !k_scale || !v_scale || !table || !cu_q || !kv_len || !out || !workspace || !status)
    return set_error(KD_ERR_ARGUMENT, "attention_cache: null pointer");
  if (total_q * (num_heads_q / num_heads_kv) > 0x7fffffff)
    return set_error(KD_ERR_ARGUMENT, "attention_cache: rows x heads per key/value head must be below 2^31");
  if (!(scale > 0.f)) return set_error(KD_ERR_ARGUMENT, "attention_cache: the scale must be positive");
  auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (!a16(q) || !a16(k_codes) || !a16(v_codes) || !a16(out) || !a16(workspace) || (gate && !a16(gate)) || ldq % 8 ||
      ldo % 8 || (gate && ldg % 8))
    return set_error(KD_ERR_ARGUMENT, "attention_cache: pointers and row strides must be 16-byte aligned");
  const int64_t wide = (int64_t)num_heads_q * head_dim;
  if (ldq < wide || ldo < wide || (gate && ldg < wide))
    return set_error(KD_ERR_ARGUMENT, "attention_cache: row strides smaller than heads x head_dim");
  ca::Args a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.gate = static_cast<const __nv_bfloat16*>(gate);
  a.ldq = ldq;
  a.ldo = ldo;
  a.ldg = ldg;
  a.table = table;
  a.ldt = ld_table;
  a.width = table_width;
  a.cu = cu_q;
  a.kv_len = kv_len;
  a.n = num_requests;
  a.total_q = total_q;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.blocks = (int)num_blocks;
  a.hq = num_heads_q;
  a.hkv = num_heads_kv;
  a.group = num_heads_q / num_heads_kv;
  a.scale_log2 = scale * 1.4426950408889634f;
  const int far = 1 << 30;  // windows past any table: sums of positions and windows stay within int32
  a.left = window_left > far ? far : window_left;
  a.right = window_right > far ? far : window_right;
  a.status = status;
  a.items = nullptr;
  a.descs = nullptr;
  a.partials = nullptr;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512)
    return set_error(KD_ERR_ARGUMENT, "attention_cache: head_dim must be 64, 128, 256 or 512");
  const int nt = ca::row_tiles_of_8(max_q, a.group, head_dim);
  if (nt == 0) return ca::row_tiles(head_dim, a, k_codes, v_codes, ws, workspace_bytes, stream);
  return ca::with_kernel(head_dim, nt, [&](auto hd, auto t) {
    return ca::launch<hd(), t()>(a, k_codes, v_codes, ws, workspace_bytes, stream);
  });
}
