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
// every (request, key/value head, 16-row tile), in that order; CTA c of P takes the tiles [c, c + 1) * total / P of
// it, so long and short requests balance to a tile without the host knowing a length. A producer warp reads 32 tiles'
// table entries and scales at a time and feeds a ring per key group by TMA; each key group (one warp, or a warp
// per 128 value columns of wide heads) takes every KG-th tile with its own running maximum and sums, and leaves a
// partial result per 16-row tile that it met; a second launch joins them.
//
// The products run on mma.sync.m16n8k16 in f16 with float32 accumulation: 16 query rows against 64 keys fit its shape
// (a 128-row tcgen05 tile would be mostly empty), and the codes turn into f16 exactly, two per conversion. Queries are
// scaled by a power of two per row (exact; f16 holds every bf16 within 2^-24 of the row's largest magnitude).
// Probabilities are rounded to f16 relative to the largest *scaled* probability p 2^e_v met (11 bits, exponents down
// to 2^-39 of it), so the blocks' value scales need no product of their own; the sum of the probabilities stays in
// float32, unrounded.
#include "cache_attention.cuh"

namespace kd {
namespace ca {

constexpr float P_SCALE = 32768.f;  // f16 probabilities hold p * 2^15 (at most 2^15; subnormal below 2^-29)

template <int HD>
struct Cfg {
  static constexpr int DV = HD < 128 ? HD : 128;  // value columns of a warp
  static constexpr int SL = HD / DV;              // warps of a key group
  static constexpr int KG = HD == 64 ? 8 : HD == 128 ? 4 : HD == 256 ? 2 : 1;  // key groups
  static constexpr int WARPS = KG * SL;
  static constexpr int THREADS = 32 * (WARPS + 1);
  static constexpr int BOX = HD < 128 ? HD : 128;  // bytes of a TMA box row (its swizzle span)
  static constexpr int CHUNKS = HD / BOX;
  static constexpr int TILE_BYTES = BN * HD;
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int STAGES = HD == 64 ? 2 : 3;
  static constexpr int Q_BYTES = RT * HD * 2;  // per key group, in fragment order
  static constexpr int SMEM = KG * (STAGES * STAGE_BYTES + Q_BYTES) + 1024 + 1024;
  static constexpr int PARTIAL = RT * (HD + 3);  // floats of one group's partial: O, then (m, M, l) per row
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

// A position in the list of key tiles: request > key/value head > 16-row tile > key tile. `advance(g)` moves forward to
// the item holding tile g.
struct Cursor {
  int i, h, rt;
  int64_t begin, end;  // the item's tiles
  int item;            // its number over the launch
  Request r;

  KD_DEVICE void load(const Args& a) {
    while (i < a.n) {
      r = request(a, i);
      if (r.nrt > 0 && r.tiles > 0) break;
      item += r.nrt * a.hkv;
      ++i;
    }
    end = begin + (i < a.n ? r.tiles : 0);
  }
  KD_DEVICE void start(const Args& a, int req, int64_t before, int items_before) {
    i = req;
    h = rt = 0;
    begin = before;
    item = items_before;
    load(a);
  }
  KD_DEVICE void seek(const Args& a, int64_t g) {
    while (i < a.n && g >= end) {
      begin = end;
      ++item;
      if (++rt == r.nrt) {
        rt = 0;
        if (++h == a.hkv) {
          h = 0;
          ++i;
          load(a);
          continue;
        }
      }
      end = begin + r.tiles;
    }
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
// d += a (16 x 16, row) * b (16 x 8, column), f16 operands, float32 sums.
KD_DEVICE void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

KD_DEVICE void group_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
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

// One tile's meta data beside its ring slot.
struct TileInfo {
  float k_scale;
  int v_exp;
  int live;  // 0: the block is absent (a table entry outside the pool): its keys are not seen
  int pad;
};

template <int HD>
__global__ void __launch_bounds__(Cfg<HD>::THREADS, 1)
    few_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Args a) {
  using C = Cfg<HD>;
  constexpr int KG = C::KG, SL = C::SL, ST = C::STAGES, DV = C::DV;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem + KG * ST * C::STAGE_BYTES;  // [KG][Q_BYTES]
  __shared__ uint64_t full[KG * ST], empty[KG * ST];
  __shared__ TileInfo info[KG * ST];
  __shared__ int64_t s_warp_tiles[C::WARPS + 1];
  __shared__ int s_warp_items[C::WARPS + 1];
  __shared__ int64_t s_lo, s_hi, s_before;
  __shared__ int s_req, s_items_before;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < KG * ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], SL);
    }
    fence_barrier_init();
  }
  // ---- this CTA's share of the tiles: a scan of the requests' tiles (twice: the total first, then the start)
  int64_t total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    const int64_t lo = pass ? total * blockIdx.x / shares(total, gridDim.x) : 0;
    int64_t carry = 0;
    int carry_items = 0;
    for (int i0 = 0; i0 < a.n; i0 += C::THREADS) {
      const int i = i0 + tid;
      int64_t w = 0;
      int items = 0;
      if (i < a.n) {
        const Request r = request(a, i);
        w = (int64_t)r.nrt * r.tiles;
        items = r.nrt;
      }
      int64_t x = w;
      int y = items;
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
      __syncthreads();
      int64_t before = carry, chunk = 0;
      int items_before = carry_items, chunk_items = 0;
#pragma unroll
      for (int v = 0; v <= C::WARPS; ++v) {
        if (v < warp) {
          before += s_warp_tiles[v];
          items_before += s_warp_items[v];
        }
        chunk += s_warp_tiles[v];
        chunk_items += s_warp_items[v];
      }
      before += x - w;
      items_before += y - items;
      if (pass && i < a.n) {
        if (blockIdx.x == 0) {  // for the launch that joins the partials
          a.tile_cu[i] = before;
          a.item_cu[i] = items_before;
        }
        if (w > 0 && lo >= before * a.hkv && lo < (before + w) * a.hkv) {
          s_req = i;
          s_before = before * a.hkv;
          s_items_before = items_before * a.hkv;
        }
      }
      carry += chunk;
      carry_items += chunk_items;
      __syncthreads();
    }
    total = carry * a.hkv;
    if (pass && tid == 0) {
      s_lo = lo;
      s_hi = blockIdx.x < shares(total, gridDim.x) ? total * (blockIdx.x + 1) / shares(total, gridDim.x) : 0;
      if (blockIdx.x == 0) {
        a.tile_cu[a.n] = carry;
        a.item_cu[a.n] = carry_items;
      }
    }
  }
  __syncthreads();
  const int64_t lo = s_lo, hi = s_hi;
  if (lo >= hi) return;

  if (warp == C::WARPS) {
    // ------------------------------------------------------------ producer
    Cursor c;
    c.start(a, s_req, s_before, s_items_before);
    if (lane == 0) {
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
    }
    // 32 tiles ahead: each lane looks up its tile's block and scales
    int64_t failed = 0;
    int z = -1, next_z = -1, ve = 0, next_ve = 0;
    float ks = 0.f, next_ks = 0.f;
    auto look_up = [&](int64_t g, int& zz, float& s, int& e) {
      zz = -1;
      s = 0.f;
      e = 0;
      if (g < hi) {
        c.seek(a, g);
        const int id = a.table[(int64_t)c.i * a.ldt + c.r.first + (int)(g - c.begin)];
        if (id >= 0 && id < a.blocks) {
          zz = id * a.hkv + c.h;
          s = a.k_scale[zz];
          e = exponent_of(a.v_scale[zz]);
        }
      }
    };
    look_up(lo + lane, next_z, next_ks, next_ve);
    for (int64_t g0 = lo; g0 < hi; g0 += 32) {
      z = next_z;
      ks = next_ks;
      ve = next_ve;
      look_up(g0 + 32 + lane, next_z, next_ks, next_ve);
      const int m = (int)min((int64_t)32, hi - g0);
      for (int j = 0; j < m; ++j) {
        const int64_t at = g0 + j - lo;
        const int zz = __shfl_sync(0xffffffffu, z, j);
        const float s = __shfl_sync(0xffffffffu, ks, j);
        const int e = __shfl_sync(0xffffffffu, ve, j);
        const int kg = (int)(at % KG);
        const int64_t use = at / KG;  // the group's tiles before this one
        const int st = kg * ST + (int)(use % ST);
        bool ok = true;
        if (lane == 0) {
          ok = mbar_wait(&empty[st], (uint32_t)((use / ST) & 1) ^ 1, a.status);
          if (ok) {
            info[st] = TileInfo{s, e, zz >= 0, 0};
            if (zz >= 0) {
              mbar_arrive_expect_tx(&full[st], C::STAGE_BYTES);
              uint8_t* dst = smem + st * C::STAGE_BYTES;
              for (int x = 0; x < C::CHUNKS; ++x) {
                tma_load_3d(&map_k, &full[st], dst + x * BN * C::BOX, x * C::BOX, 0, zz);
                tma_load_3d(&map_v, &full[st], dst + C::TILE_BYTES + x * BN * C::BOX, x * C::BOX, 0, zz);
              }
            } else {
              mbar_arrive(&full[st]);
            }
          }
        }
        if (!__shfl_sync(0xffffffffu, ok, 0)) {
          failed = at;
          goto drain;
        }
      }
    }
    return;
  drain:
    // A consumer gave up: wait (bounded) for the copies in flight before the shared memory goes away. Tiles before
    // `failed` were issued; slot (kg, st) last took its group's tile u.
    if (lane == 0) {
      const uint64_t start = globaltimer();
      for (int s = 0; s < KG * ST; ++s) {
        const int64_t issued = (failed - s / ST + KG - 1) / KG;
        const int64_t u = issued - 1 - ((issued - 1 - s % ST) % ST + ST) % ST;
        if (u < 0) continue;
        while (!mbar_try_wait(smem_u32(&full[s]), (uint32_t)((u / ST) & 1)) && globaltimer() - start < 1000000000ull) {
        }
      }
    }
    return;
  }

  // ------------------------------------------------------------ consumers
  const int kg = warp / SL, slice = warp % SL;
  const int row_a = lane >> 2, t4 = lane & 3;  // this thread's rows are row_a and row_a + 8 of the 16-row tile
  uint4* qf = reinterpret_cast<uint4*>(s_q + kg * C::Q_BYTES);
  const uint32_t ring = smem_u32(smem) + kg * ST * C::STAGE_BYTES;
  Cursor c;
  c.start(a, s_req, s_before, s_items_before);
  c.seek(a, lo);
  int64_t use = 0;    // the group's tiles so far
  bool dead = false;  // a wait gave up: walk on to the end without computing, so that no warp waits at a barrier alone
  for (int64_t g = lo; g < hi;) {
    const int64_t stop = min(c.end, hi);  // the fragment of this item: tiles [g, stop)
    const int rows = min(RT, c.r.lq * a.group - c.rt * RT);
    // ---- queries: f16, scaled to the row's largest magnitude, in the order of the A fragments
    float q_scale[2];
    const __nv_bfloat16* qp[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = c.rt * RT + row_a + 8 * u;
      const bool live = row_a + 8 * u < rows;
      const int tok = live ? r / a.group : 0;
      qp[u] = live ? a.q + (int64_t)(c.r.q0 + tok) * a.ldq + (c.h * a.group + r - tok * a.group) * HD + 4 * t4 : nullptr;
    }
    if (SL > 1) group_sync(1 + kg, SL * 32);  // the previous item's queries have been read
    else __syncwarp();
    {
      uint32_t big[2] = {0, 0};  // the largest finite magnitude as a bf16 pattern
#pragma unroll 4
      for (int x = 0; x < HD / 16; ++x)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint2 w = qp[u] ? *reinterpret_cast<const uint2*>(qp[u] + 16 * x) : make_uint2(0, 0);
          const uint32_t v[4] = {w.x & 0x7fffu, (w.x >> 16) & 0x7fffu, w.y & 0x7fffu, (w.y >> 16) & 0x7fffu};
#pragma unroll
          for (int e = 0; e < 4; ++e) big[u] = max(big[u], v[e] < 0x7f80u ? v[e] : 0u);
        }
      float inv[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        big[u] = max(big[u], __shfl_xor_sync(0xffffffffu, big[u], 1));
        big[u] = max(big[u], __shfl_xor_sync(0xffffffffu, big[u], 2));
        const int e = max((int)(big[u] >> 7) - 127, -120);
        q_scale[u] = pow2i(e);
        inv[u] = pow2i(-e);
      }
#pragma unroll 4
      for (int x = slice; x < HD / 16; x += SL) {
        uint4 f;
        const uint2 w0 = qp[0] ? *reinterpret_cast<const uint2*>(qp[0] + 16 * x) : make_uint2(0, 0);
        const uint2 w1 = qp[1] ? *reinterpret_cast<const uint2*>(qp[1] + 16 * x) : make_uint2(0, 0);
        float2 p = unpack_bf16x2(w0.x), r = unpack_bf16x2(w0.y);
        f.x = pack_f16x2(p.x * inv[0], p.y * inv[0]);
        f.z = pack_f16x2(r.x * inv[0], r.y * inv[0]);
        p = unpack_bf16x2(w1.x);
        r = unpack_bf16x2(w1.y);
        f.y = pack_f16x2(p.x * inv[1], p.y * inv[1]);
        f.w = pack_f16x2(r.x * inv[1], r.y * inv[1]);
        qf[x * 32 + lane] = f;
      }
    }
    if (SL > 1) group_sync(1 + kg, SL * 32);
    else __syncwarp();
    // the rows' visible keys
    int key_lo[2], key_hi[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = c.rt * RT + row_a + 8 * u;
      const int pos = r / a.group + c.r.lk - c.r.lq;
      key_lo[u] = a.left >= 0 ? pos - a.left : 0;
      key_hi[u] = a.right >= 0 ? min(c.r.lk - 1, pos + a.right) : c.r.lk - 1;
    }
    // the tile's rows from the first to the last: which key tiles need a mask
    const int pos0 = c.rt * RT / a.group + c.r.lk - c.r.lq;
    const int pos1 = (c.rt * RT + rows - 1) / a.group + c.r.lk - c.r.lq;

    float m[2] = {-INFINITY, -INFINITY};  // running maximum of x (log2 units)
    float big[2] = {-INFINITY, -INFINITY};  // running maximum of x + e_v
    float l[2] = {0.f, 0.f};
    float o[DV / 8][4];
#pragma unroll
    for (int d = 0; d < DV / 8; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] = 0.f;

    for (int64_t t = g + ((kg - (g - lo)) % KG + KG) % KG; t < stop; t += KG, ++use) {
      const int st = (int)(use % ST);
      dead = dead || !mbar_wait(&full[kg * ST + st], (uint32_t)((use / ST) & 1), a.status);
      if (__any_sync(0xffffffffu, dead)) {
        dead = true;
        continue;
      }
      const TileInfo ti = info[kg * ST + st];
      const uint32_t sk = ring + st * C::STAGE_BYTES, sv = sk + C::TILE_BYTES;
      if (ti.live) {
        // ---- S = Q K^T: 8 n-tiles of 8 keys; thread (row_a, t4) holds keys 8 j + 2 t4, + 1 of its two rows
        float s[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll 8
        for (int x = 0; x < HD / 16; ++x) {
          const uint4 f = qf[x * 32 + lane];
          const uint32_t af[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t w[4];
            ldmatrix4(sk + piece<HD>(half * 32 + lane, x), w);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              uint32_t b0, b1;
              codes_to_f16(w[y], b0, b1);
              mma_f16(s[half * 4 + y], af, b0, b1);
            }
          }
        }
        const int key0 = (c.r.first + (int)(t - c.begin)) * BN;
        const bool tail = key0 + BN > c.r.lk;  // rows past the request's tokens hold anything
        const bool edge = tail || (a.right >= 0 && key0 + BN - 1 > pos0 + a.right) || (a.left >= 0 && key0 < pos1 - a.left);
        // ---- softmax: two rows, 16 keys each, over the quad's four threads
        float factor[2], alpha_o[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float mul = score_factor(q_scale[u] * a.scale_log2, ti.k_scale);
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = s[j][2 * u + e] * mul;
              if (edge) {
                const int key = key0 + 8 * j + 2 * t4 + e;
                x = key >= key_lo[u] && key <= key_hi[u] ? x : -INFINITY;
              }
              s[j][2 * u + e] = x;
              mx = fmaxf(mx, x);
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m[u], mx), big_new = fmaxf(big[u], mx + (float)ti.v_exp);
          const float base = m_new == -INFINITY ? 0.f : m_new, vbase = big_new == -INFINITY ? 0.f : big_new;
          const float alpha = fast_exp2(m[u] - base);  // 0 while nothing was seen
          alpha_o[u] = fast_exp2(big[u] - vbase);
          factor[u] = fast_exp2(fminf(base - vbase + (float)ti.v_exp, 110.f)) * P_SCALE;
          m[u] = m_new;
          big[u] = big_new;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float p = fast_exp2(s[j][2 * u + e] - base);
              sum += p;
              s[j][2 * u + e] = p * factor[u];
            }
          l[u] = l[u] * alpha + sum;
        }
#pragma unroll
        for (int d = 0; d < DV / 8; ++d) {
          o[d][0] *= alpha_o[0];
          o[d][1] *= alpha_o[0];
          o[d][2] *= alpha_o[1];
          o[d][3] *= alpha_o[1];
        }
        // ---- O += P V: 16 keys per step; two n-tiles per 16 value columns, the even and the odd ones
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint32_t pf[4] = {pack_f16x2(s[2 * kk][0], s[2 * kk][1]), pack_f16x2(s[2 * kk][2], s[2 * kk][3]),
                                  pack_f16x2(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                                  pack_f16x2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
          // codes of keys past the request's last token are cleared: a probability of 0 times a NaN code is NaN
          uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
          if (tail) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int left_keys = c.r.lk - (key0 + kk * 16 + y * 8 + 2 * t4);
              keep[y] = left_keys >= 2 ? 0xffffffffu : left_keys == 1 ? 0x0000ffffu : 0u;
            }
          }
#pragma unroll
          for (int x = 0; x < DV / 32; ++x) {
            uint32_t w[4];  // (keys 0-7, keys 8-15) of 16-column piece 2 x, then of 2 x + 1
            ldmatrix4_trans(sv + piece<HD>(kk * 16 + (lane & 15), slice * (DV / 16) + 2 * x + (lane >> 4)), w);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t a0, a1, b0, b1;  // (even, odd columns) of keys 0-7 and of keys 8-15
              codes_to_f16(__byte_perm(w[2 * y] & keep[0], 0, 0x3120), a0, a1);
              codes_to_f16(__byte_perm(w[2 * y + 1] & keep[1], 0, 0x3120), b0, b1);
              mma_f16(o[(2 * x + y) * 2], pf, a0, b0);
              mma_f16(o[(2 * x + y) * 2 + 1], pf, a1, b1);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[kg * ST + st]);
    }
    // ---- the group's partial of this fragment: item + CTA number its place (both only grow along the list)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
    }
    float* part = a.partials + ((int64_t)(c.item + (int)blockIdx.x) * KG + kg) * C::PARTIAL;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = row_a + 8 * u;
      if (r < rows) {
        if (slice == 0 && t4 == 0) {
          float* st3 = part + RT * HD + 3 * r;
          st3[0] = m[u];
          st3[1] = big[u];
          st3[2] = l[u];
        }
        if (big[u] != -INFINITY || l[u] != 0.f) {
#pragma unroll
          for (int x = 0; x < DV / 16; ++x)
            *reinterpret_cast<float4*>(part + r * HD + slice * DV + 16 * x + 4 * t4) =
                make_float4(o[2 * x][2 * u], o[2 * x + 1][2 * u], o[2 * x][2 * u + 1], o[2 * x + 1][2 * u + 1]);
        }
      }
    }
    g = stop;
    c.seek(a, g);
  }
}

// Joins the partials of one row of one item: blockIdx.x the item, blockIdx.y its row. Every partial's (m, M, l) is
// read twice and its O once; partials lie in the order of the keys, and so do the sums.
template <int HD>
__global__ void __launch_bounds__(128) join_kernel(Args a, int ctas) {
  using C = Cfg<HD>;
  constexpr int V = HD / 64 < 4 ? HD / 64 : 4;  // columns a thread holds at once
  constexpr int LANES = HD / V < 128 ? HD / V : 128;
  constexpr int GROUPS = 128 / LANES;           // partials taken at once
  constexpr int PASSES = HD / (V * LANES);
  const int item = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  if (item >= a.item_cu[a.n] * a.hkv) return;
  int lo = 0, hi = a.n - 1;  // the request holding the item
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if ((int64_t)a.item_cu[mid] * a.hkv <= item)
      lo = mid;
    else
      hi = mid - 1;
  }
  const Request r = request(a, lo);
  const int local = item - a.item_cu[lo] * a.hkv;
  const int h = local / r.nrt, rt = local - h * r.nrt;
  const int gr = rt * RT + row;
  if (gr >= r.lq * a.group) return;
  const int tok = gr / a.group;
  const int head = h * a.group + gr - tok * a.group;
  const int64_t total = a.tile_cu[a.n] * a.hkv;
  const int64_t begin = a.tile_cu[lo] * a.hkv + (int64_t)local * r.tiles, end = begin + r.tiles;
  // CTA c holds tiles [c total / P, (c + 1) total / P): the one holding tile g is ((g + 1) P - 1) / total
  const int64_t p = shares(total, ctas);
  const int c0 = r.tiles ? (int)(((begin + 1) * p - 1) / total) : 0;
  const int c1 = r.tiles ? (int)((end * p - 1) / total) : -1;
  const int n = (c1 - c0 + 1) * C::KG;
  const float* part = a.partials + (int64_t)(item + c0) * C::KG * C::PARTIAL;
  __shared__ float s_red[3][4];
  float m = -INFINITY, big = -INFINITY;
  for (int p = tid; p < n; p += 128) {
    const float* st3 = part + (int64_t)p * C::PARTIAL + RT * HD + 3 * row;
    m = fmaxf(m, st3[0]);
    big = fmaxf(big, st3[1]);
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
  }
  if ((tid & 31) == 0) {
    s_red[0][tid / 32] = m;
    s_red[1][tid / 32] = big;
  }
  __syncthreads();
  m = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
  big = fmaxf(fmaxf(s_red[1][0], s_red[1][1]), fmaxf(s_red[1][2], s_red[1][3]));
  const float base = m == -INFINITY ? 0.f : m, vbase = big == -INFINITY ? 0.f : big;
  float l = 0.f;
  for (int p = tid; p < n; p += 128) {
    const float* st3 = part + (int64_t)p * C::PARTIAL + RT * HD + 3 * row;
    l += st3[2] * fast_exp2(st3[0] - base);
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  if ((tid & 31) == 0) s_red[2][tid / 32] = l;
  __syncthreads();
  l = (s_red[2][0] + s_red[2][1]) + (s_red[2][2] + s_red[2][3]);
  // o = O 2^(M - m) / (2^15 l); without a visible key 0
  const float fin = l == 0.f ? 0.f : fast_exp2(fminf(vbase - base, 126.f)) / (l * P_SCALE);
  __shared__ float s_o[GROUPS > 1 ? 128 * V : 1];
  const int grp = tid / LANES, col = (tid % LANES) * V;
  const int64_t orow = (int64_t)(r.q0 + tok) * a.ldo + (int64_t)head * HD;
  const int64_t grow = (int64_t)(r.q0 + tok) * a.ldg + (int64_t)head * HD;
#pragma unroll
  for (int pass = 0; pass < PASSES; ++pass) {
    const int cc = col + pass * V * LANES;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    for (int p = grp; p < n; p += GROUPS) {
      const float* pp = part + (int64_t)p * C::PARTIAL;
      const float st_big = pp[RT * HD + 3 * row + 1];
      if (st_big == -INFINITY && pp[RT * HD + 3 * row + 2] == 0.f) continue;  // this group met no key of the row
      const float w = fast_exp2(st_big - vbase);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += w * pp[row * HD + cc + e];
    }
    if constexpr (GROUPS > 1) {
#pragma unroll
      for (int e = 0; e < V; ++e) s_o[tid * V + e] = acc[e];
      __syncthreads();
      if (grp == 0) {
#pragma unroll
        for (int gq = 1; gq < GROUPS; ++gq)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += s_o[(gq * LANES + tid) * V + e];
      }
    }
    if (grp == 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float x = l == 0.f ? 0.f : acc[e] * fin;
        if (a.gate && l != 0.f) x *= sigmoid(__bfloat162float(a.gate[grow + cc + e]));
        a.out[orow + cc + e] = __float2bfloat16_rn(x);
      }
    }
  }
}

// Whether the requests' rows per key/value head fit one 16-row tile: the kernel of this file. Both kernels are right for
// any rows.
static bool few_rows(int max_q, int group) { return (int64_t)max_q * group <= RT; }

// Bytes of scratch: the two request arrays, then one partial per (item + CTA, key group).
template <int HD>
int64_t few_rows_items(int n, int64_t total_q, int hkv, int group) {
  return ((total_q * group + RT - 1) / RT + n) * hkv;
}
int64_t header_bytes(int n) { return ((int64_t)(n + 1) * 12 + 15) / 16 * 16 + 16; }

template <int HD>
int64_t workspace_bytes(int n, int64_t total_q, int hkv, int group, int ctas) {
  return header_bytes(n) +
         (few_rows_items<HD>(n, total_q, hkv, group) + ctas) * Cfg<HD>::KG * Cfg<HD>::PARTIAL * (int64_t)sizeof(float);
}

template <int HD>
int launch(Args a, const void* k_codes, const void* v_codes, uint8_t* ws, int64_t ws_bytes, cudaStream_t stream) {
  using C = Cfg<HD>;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(KD_ERR_ARGUMENT, "attention_cache: device index");
  const int ctas = num_sms(dev);
  const int64_t items = few_rows_items<HD>(a.n, a.total_q, a.hkv, a.group);
  if (items > 0x7fffffff - 4096) return set_error(KD_ERR_ARGUMENT, "attention_cache: too many row tiles");
  if (ws_bytes < workspace_bytes<HD>(a.n, a.total_q, a.hkv, a.group, ctas))
    return set_error(KD_ERR_ARGUMENT, "attention_cache: workspace smaller than kd_attention_cache_workspace");
  a.tile_cu = reinterpret_cast<int64_t*>(ws);
  a.item_cu = reinterpret_cast<int32_t*>(ws + 8 * (int64_t)(a.n + 1));
  a.partials = reinterpret_cast<float*>(ws + header_bytes(a.n));
  CUtensorMap mk, mv;
  const auto dt = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const auto sw = HD == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  int rc = make_tma_3d(&mk, k_codes, dt, 1, HD, BN, (uint64_t)a.blocks * a.hkv, HD, (uint64_t)BN * HD, C::BOX, BN, 1,
                       sw);
  if (!rc)
    rc = make_tma_3d(&mv, v_codes, dt, 1, HD, BN, (uint64_t)a.blocks * a.hkv, HD, (uint64_t)BN * HD, C::BOX, BN, 1, sw);
  if (rc) return rc;
  auto kernel = few_rows_kernel<HD>;
  static bool configured[64] = {false};
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return record_cuda_error(e, "attention_cache: cudaFuncSetAttribute");
    configured[dev] = true;
  }
  kernel<<<ctas, C::THREADS, C::SMEM, stream>>>(mk, mv, a);
  rc = record_cuda_error(cudaGetLastError(), "attention_cache: launch");
  if (rc) return rc;
  join_kernel<HD><<<dim3((unsigned)items, RT), 128, 0, stream>>>(a, ctas);
  return record_cuda_error(cudaGetLastError(), "attention_cache: join launch");
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
  if (!ca::few_rows(max_q, group)) {
    *bytes = ca::row_tiles_workspace(head_dim, sms);
    return KD_OK;
  }
  switch (head_dim) {
    case 64: *bytes = ca::workspace_bytes<64>(num_requests, total_q, num_heads_kv, group, sms); break;
    case 128: *bytes = ca::workspace_bytes<128>(num_requests, total_q, num_heads_kv, group, sms); break;
    case 256: *bytes = ca::workspace_bytes<256>(num_requests, total_q, num_heads_kv, group, sms); break;
    default: *bytes = ca::workspace_bytes<512>(num_requests, total_q, num_heads_kv, group, sms); break;
  }
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
  a.tile_cu = nullptr;
  a.item_cu = nullptr;
  a.partials = nullptr;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512)
    return set_error(KD_ERR_ARGUMENT, "attention_cache: head_dim must be 64, 128, 256 or 512");
  if (!ca::few_rows(max_q, a.group)) return ca::row_tiles(head_dim, a, k_codes, v_codes, ws, workspace_bytes, stream);
  switch (head_dim) {
    case 64: return ca::launch<64>(a, k_codes, v_codes, ws, workspace_bytes, stream);
    case 128: return ca::launch<128>(a, k_codes, v_codes, ws, workspace_bytes, stream);
    case 256: return ca::launch<256>(a, k_codes, v_codes, ws, workspace_bytes, stream);
    default: return ca::launch<512>(a, k_codes, v_codes, ws, workspace_bytes, stream);
  }
}
