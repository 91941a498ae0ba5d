// A cache of states: block tables and slot maps from request lengths, and the write of keys and values into blocks of
// e4m3 codes with one power-of-two scale per (block, key/value head). The attention over the blocks is in
// cache_attention.cu.
//
// One block holds KD_KV_BLOCK = 64 tokens of one request. Scales are powers of two: the codes' relative precision does
// not depend on the scale (e4m3 is a floating-point format), a code times its scale is exact in bf16 and f16 scaled by
// an exponent, and a block whose scale grows while it fills keeps its old codes exactly except where they turn
// subnormal. There is no counterpart in the reference, which computes every request from its first token.
#include "common.cuh"
#include "kd_internal.h"

namespace kd {
namespace kv {

constexpr int BLOCK = KD_KV_BLOCK;
constexpr int TABLE_THREADS = 1024;
constexpr int MAX_REQUESTS = 16384;  // the per-request arrays of the table kernels live in shared memory

KD_DEVICE int blocks_of(int tokens) { return (int)(((int64_t)tokens + BLOCK - 1) / BLOCK); }

// Exclusive sum of `v` over the block's threads (every thread gets its own prefix) and the total.
KD_DEVICE int block_exclusive_sum(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = lane < (int)blockDim.x / 32 ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const int before = warp == 0 ? 0 : warp_sums[warp - 1];
  total = warp_sums[31];
  __syncthreads();
  return before + x - v;
}

KD_DEVICE bool in_pool(int id, int capacity) { return (uint32_t)id < (uint32_t)capacity; }

// Ids met so far, a bit each: SEEN_BLOCKS ids from `from` on at a time (one pass for pools up to that size, so that
// nothing waits for it), in shared memory.
constexpr int SEEN_BLOCKS = 1 << 18;
__host__ __device__ constexpr int seen_words(int capacity) {
  return (capacity < SEEN_BLOCKS ? capacity : SEEN_BLOCKS) / 32 + 1;
}
// Marks an id of the pool; whether it was marked before.
KD_DEVICE bool met_before(uint32_t* seen, int id, int from) {
  const uint32_t at = (uint32_t)id - (uint32_t)from;
  if (at >= (uint32_t)SEEN_BLOCKS) return false;
  return (atomicOr(&seen[at / 32], 1u << (at & 31)) >> (at & 31)) & 1u;
}

// The last i in [0, n) with keys[i] <= x (keys ascending, keys[0] <= x).
KD_DEVICE int last_at_most(const int* keys, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (keys[mid] <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// ------------------------------------------------------------------------------------------------ block tables

struct AssignArgs {
  const int32_t* lens;
  const int32_t* cu;
  int n;
  int64_t rows;
  int32_t* table;
  int64_t ldt;
  int width;
  const int32_t* free_ids;
  int capacity;
  int32_t* count;  // [0] free blocks, [1] the outcome
  int32_t* kv_len;
  int64_t* seqpos;
  int64_t* slots;
};

// One cluster of 1-8 CTAs, each scanning every request's new blocks on its own (a few thousand integers in L2), then
// taking its share of the rows. The k-th new block of the launch is the k-th from the top of the free stack, so every
// CTA knows the new blocks without reading the table that others write; a new block's table entry is written by the
// thread of the block's first row. The stack's count and kv_len (which may be `lens` itself)
// change after a cluster barrier, when every CTA has read them. Every CTA also looks at the ids that the rows will use,
// the half-filled blocks' table entries during the scan and the new blocks' on the stack after it: one outside the pool,
// or one met twice, whose rows two requests would write, refuses the call before anything is written.
// Bound by latency: dependent reads of the lengths, of the stack and of the table, and the launch. With the release after
// it, as graph replays: one request 7.5 us, 512 requests of 45,473 rows 15.1 us (0.6 of each for the ids' checks).
__global__ void __launch_bounds__(TABLE_THREADS) assign_kernel(AssignArgs a) {
  extern __shared__ int smem[];
  int* s_cu = smem;                // [n + 1]
  int* s_len = s_cu + a.n + 1;     // [n]
  int* s_base = s_len + a.n;       // [n]: the request's first new block, counted over the launch
  uint32_t* s_seen = reinterpret_cast<uint32_t*>(s_base + a.n);  // [seen_words]
  const int words = seen_words(a.capacity);
  __shared__ int warp_sums[32];
  __shared__ int s_bad;
  const int tid = threadIdx.x;
  if (tid == 0) s_bad = 0;
  const int have_free = a.count[0];
  for (int i = tid; i <= a.n; i += TABLE_THREADS) s_cu[i] = a.cu[i];
  for (int i = tid; i < a.n; i += TABLE_THREADS) s_len[i] = a.lens[i];
  for (int w = tid; w < words; w += TABLE_THREADS) s_seen[w] = 0;
  const bool stack_ok = have_free >= 0 && have_free <= a.capacity;
  const int top = stack_ok && tid < have_free ? a.free_ids[have_free - 1 - tid] : -1;  // here when the scan is done
  __syncthreads();
  int carry = 0;
  for (int i0 = 0; i0 < a.n; i0 += TABLE_THREADS) {
    const int i = i0 + tid;
    int add = 0, part = -1;
    bool half = false;  // new rows go on in the half-filled block `part`
    if (i < a.n) {
      const int len = s_len[i];
      const int64_t grown = (int64_t)s_cu[i + 1] - s_cu[i];
      const bool malformed = len < 0 || grown < 0 || s_cu[i] < 0 || s_cu[i + 1] > a.rows || len + grown > 0x7fffffff;
      if (malformed) {
        atomicMin(&s_bad, KD_KV_MALFORMED);
      } else if ((len + grown + BLOCK - 1) / BLOCK > a.width) {
        atomicMin(&s_bad, KD_KV_TABLE_FULL);
      } else {
        add = (int)((len + grown + BLOCK - 1) / BLOCK) - blocks_of(len);
        half = grown > 0 && len % BLOCK > 0;
        if (half) part = a.table[(int64_t)i * a.ldt + len / BLOCK];
      }
    }
    int total;
    const int base = block_exclusive_sum(add, warp_sums, total);
    if (i < a.n) s_base[i] = carry + base;
    if (half && (!in_pool(part, a.capacity) || met_before(s_seen, part, 0))) atomicMin(&s_bad, KD_KV_MALFORMED);
    carry += total;
  }
  const int needed = carry;
  if (stack_ok && needed <= have_free) {
    for (int j = tid; j < needed; j += TABLE_THREADS) {
      const int id = j < TABLE_THREADS ? top : a.free_ids[have_free - 1 - j];
      if (!in_pool(id, a.capacity) || met_before(s_seen, id, 0)) atomicMin(&s_bad, KD_KV_MALFORMED);
    }
  }
  __syncthreads();
  if (a.capacity > SEEN_BLOCKS && s_bad == 0 && stack_ok && needed <= have_free) {  // the ids past the first pass's
    for (int from = SEEN_BLOCKS; from < a.capacity && from > 0; from += SEEN_BLOCKS) {
      __syncthreads();
      for (int w = tid; w < words; w += TABLE_THREADS) s_seen[w] = 0;
      __syncthreads();
      bool twice = false;
      for (int i = tid; i < a.n; i += TABLE_THREADS)
        if (s_cu[i + 1] > s_cu[i] && s_len[i] % BLOCK > 0)
          twice |= met_before(s_seen, a.table[(int64_t)i * a.ldt + s_len[i] / BLOCK], from);
      for (int j = tid; j < needed; j += TABLE_THREADS) twice |= met_before(s_seen, a.free_ids[have_free - 1 - j], from);
      if (__syncthreads_or(twice)) {
        if (tid == 0) s_bad = KD_KV_MALFORMED;
        break;
      }
    }
    __syncthreads();
  }
  const int bad = !stack_ok ? KD_KV_MALFORMED : s_bad;
  const bool ok = bad == 0 && needed <= have_free;
  const bool positions = bad != KD_KV_MALFORMED;

  const int64_t step = (int64_t)gridDim.x * TABLE_THREADS;
  const int first = a.n > 0 ? s_cu[0] : 0, last = a.n > 0 ? s_cu[a.n] : 0;
  for (int64_t t = (int64_t)blockIdx.x * TABLE_THREADS + tid; t < a.rows; t += step) {
    int64_t slot = -1, pos = 0;
    if (positions && t >= first && t < last) {
      const int i = last_at_most(s_cu, a.n, (int)t);
      const int len = s_len[i];
      pos = len + (t - s_cu[i]);
      if (ok) {
        const int b = (int)(pos / BLOCK), had = blocks_of(len);
        int id;
        if (b < had) {
          id = a.table[(int64_t)i * a.ldt + b];
        } else {
          id = a.free_ids[have_free - 1 - (s_base[i] + b - had)];
          if (pos % BLOCK == 0) a.table[(int64_t)i * a.ldt + b] = id;
        }
        slot = (int64_t)id * BLOCK + pos % BLOCK;
      }
    }
    a.seqpos[t] = pos;
    a.slots[t] = slot;
  }
  cluster_sync();
  if (blockIdx.x == 0) {
    for (int i = tid; i < a.n; i += TABLE_THREADS) a.kv_len[i] = s_len[i] + (ok ? s_cu[i + 1] - s_cu[i] : 0);
    if (tid == 0) {
      if (ok) a.count[0] = have_free - needed;
      a.count[1] = bad != 0 ? bad : ok ? 0 : needed - have_free;
    }
  }
}

struct ReleaseArgs {
  int32_t* table;
  int64_t ldt;
  int width;
  const int32_t* lens;
  const int32_t* keep;
  int n;
  int32_t* free_ids;
  int capacity;
  int32_t* count;
};

// The blocks past each request's first `keep` tokens go back on the stack, the last request's last block first: an
// assignment followed by its release leaves the stack as it was. One CTA: the first pass checks every entry, so a table
// with an id outside the pool, or with one named twice among those given back, gives nothing back. The outcome word keeps
// what the assignment before it left there, so that a failure survives the sequence of one step.
__global__ void __launch_bounds__(TABLE_THREADS) release_kernel(ReleaseArgs a) {
  extern __shared__ int smem[];
  int* s_base = smem;           // [n]
  int* s_from = s_base + a.n;   // [n]: the first block given back
  uint32_t* s_seen = reinterpret_cast<uint32_t*>(s_from + a.n);  // [seen_words]
  const int words = seen_words(a.capacity);
  __shared__ int warp_sums[32];
  __shared__ int s_bad;
  const int tid = threadIdx.x;
  if (tid == 0) s_bad = 0;
  const int have_free = a.count[0];
  for (int w = tid; w < words; w += TABLE_THREADS) s_seen[w] = 0;
  __syncthreads();
  int carry = 0;
  for (int i0 = 0; i0 < a.n; i0 += TABLE_THREADS) {
    const int i = i0 + tid;
    int drop = 0;
    if (i < a.n) {
      const int len = a.lens[i], kept = min(max(a.keep[i], 0), max(len, 0));
      if (len < 0 || blocks_of(len) > a.width) {
        atomicMin(&s_bad, KD_KV_MALFORMED);
      } else {
        s_from[i] = blocks_of(kept);
        drop = blocks_of(len) - s_from[i];
      }
    }
    int total;
    const int base = block_exclusive_sum(drop, warp_sums, total);
    if (i < a.n) s_base[i] = carry + base;
    carry += total;
  }
  __syncthreads();
  const int dropped = carry;
  const bool sized = s_bad == 0 && have_free >= 0 && (int64_t)have_free + dropped <= a.capacity;
  if (sized) {
    for (int from = 0; from < a.capacity && from >= 0; from += SEEN_BLOCKS) {
      if (from > 0) {
        for (int w = tid; w < words; w += TABLE_THREADS) s_seen[w] = 0;
        __syncthreads();
      }
      for (int j = tid; j < dropped; j += TABLE_THREADS) {
        const int i = last_at_most(s_base, a.n, j);
        const int id = a.table[(int64_t)i * a.ldt + s_from[i] + j - s_base[i]];
        if (!in_pool(id, a.capacity) || met_before(s_seen, id, from)) atomicMin(&s_bad, KD_KV_MALFORMED);
      }
      __syncthreads();
    }
  }
  const bool ok = sized && s_bad == 0;
  if (ok) {
    for (int j = tid; j < dropped; j += TABLE_THREADS) {
      const int i = last_at_most(s_base, a.n, j);
      int32_t* entry = a.table + (int64_t)i * a.ldt + s_from[i] + j - s_base[i];
      a.free_ids[have_free + dropped - 1 - j] = *entry;
      *entry = -1;
    }
  }
  if (tid == 0) {
    if (ok)
      a.count[0] = have_free + dropped;
    else
      a.count[1] = KD_KV_MALFORMED;
  }
}

// ------------------------------------------------------------------------------------------------ the write

constexpr int store_threads(int head_dim) { return 2 * head_dim; }  // a thread holds 4 pieces of k and of v
constexpr int E_MIN = -100, E_MAX = 120;  // the scales' exponents (E_MAX holds the largest bf16 value)

// The least exponent e with a 2^-e <= 448 = 1.75 * 2^8, within [E_MIN, E_MAX]; a >= 0, finite.
KD_DEVICE int scale_exponent(float a) {
  const uint32_t u = __float_as_uint(a);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, E_MIN), E_MAX);
}

KD_DEVICE float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // e in [-126, 127]

struct StoreArgs {
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t ldk, ldv, rows;
  const int32_t* cu;
  int n, heads;
  const int64_t* slots;
  int64_t blocks;
  uint8_t* k_codes;
  uint8_t* v_codes;
  float* k_scale;
  float* v_scale;
};

// Two values as packed e4m3 codes, round to nearest even, saturating at +-448; NaN stays NaN.
KD_DEVICE uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
KD_DEVICE float2 from_e4m3x2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

KD_DEVICE uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("max.u16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
// The larger of the even and of the odd elements' magnitudes.
KD_DEVICE uint32_t largest(const uint4& x) {
  return max_u16x2(max_u16x2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), max_u16x2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
}
// Raises `top` to the largest finite magnitude's pattern; whether there is a NaN.
KD_DEVICE bool finite_max(const uint4& x, uint32_t& top) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  bool nan = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t y = (w[e / 2] >> (16 * (e & 1))) & 0x7fffu;
    nan |= y > 0x7f80u;
    top = max(top, y < 0x7f80u ? y : 0u);
  }
  return nan;
}

// One CTA writes the new rows of one block for one key/value head: loads them (16 bytes a thread and step, all loads in
// flight at once), takes the largest finite magnitude of the keys and of the values, and writes codes of 8 bytes a
// thread, so that a row of 128 codes is one line. A block whose first new row is not its first row keeps the larger of
// its old scale and the new rows' own; where it grows, the old codes are brought to it (code * 2^(old - new), rounded
// to nearest even). Requests' blocks are laid over the grid by f(i) = cu[i] / 64 + 2 i, which leaves every request
// enough places (its rows touch at most rows / 64 + 2 blocks) without a scan; each warp finds its request by probing 32
// requests at a time.
//
// Bound by the reads of k and v, next to it by the instructions per element (magnitudes as two 16-bit integers to a
// word, elements one by one only where one is not finite: 46.5 -> 38 us), then by the loads in flight: for heads of 64
// and 128 1,280 threads an SM at 48 registers (38 -> 35.9 us; at 40 they spill, 40 us), for heads of 256 and 512 the
// two and the one CTA that fit, 1,024. 33,349 rows of 8 heads of 128 (205 MB): 36.1 us, 5.68 TB/s; as many bytes in 16
// heads of 64 39 us, in 4 of 256 41 us, in 2 of 512 52 us. One CTA with several heads one after another, the next
// one's loads in flight, was slower (39 us), as were neighbouring heads first. The smallest launches are a chain of
// dependent loads, 6.1 us.
template <int HD>
__global__ void __launch_bounds__(store_threads(HD), 1280 / store_threads(HD))
    store_kernel(StoreArgs a) {
  constexpr int THREADS = store_threads(HD);
  constexpr int VEC = HD / 8;                            // 8-element pieces of a row
  constexpr int STEPS = BLOCK * VEC / THREADS;     // pieces a thread holds of k and of v
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int64_t place = blockIdx.x;
  // the last request i with f(i) <= place
  int lo = 0, count = a.n;
  while (count > 1) {
    const int step = (count + 31) / 32;
    const int i = lo + min(lane * step, count - 1);
    const bool at_most = (int64_t)(a.cu[i] / BLOCK) + 2 * (int64_t)i <= place;
    const int hits = __popc(__ballot_sync(0xffffffffu, at_most));  // f ascends: lanes 0 .. hits - 1
    const int skip = max(hits - 1, 0) * step;
    const int next = min(skip, count - 1);
    count = min(step, count - next);
    lo += next;
  }
  const int req = lo;
  const int64_t first = a.cu[req], end = a.cu[req + 1];
  const int64_t j = place - (first / BLOCK + 2 * (int64_t)req);
  if (first < 0 || end > a.rows || end <= first || j < 0) return;
  const int64_t slot0 = a.slots[first];
  if (slot0 < 0) return;
  const int head_part = BLOCK - (int)(slot0 % BLOCK);  // rows of the request's first block
  const int64_t row0 = j == 0 ? first : first + head_part + (j - 1) * BLOCK;
  if (row0 >= end) return;
  const int64_t slot = j == 0 ? slot0 : a.slots[row0];
  if (slot < 0 || slot >= a.blocks * BLOCK) return;
  const int64_t block = slot / BLOCK;
  const int off = (int)(slot % BLOCK);
  const int live = (int)min((int64_t)(BLOCK - off), end - row0);
  const int head = blockIdx.y;

  const int64_t at = block * a.heads + head;
  float old_scale[2] = {};
  if (off > 0) {
    old_scale[0] = a.k_scale[at];
    old_scale[1] = a.v_scale[at];
  }
  uint4 kx[STEPS], vx[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int p = s * THREADS + threadIdx.x, r = p / VEC, c = (p % VEC) * 8;
    if (r < live) {
      kx[s] = *reinterpret_cast<const uint4*>(a.k + (row0 + r) * a.ldk + head * HD + c);
      vx[s] = *reinterpret_cast<const uint4*>(a.v + (row0 + r) * a.ldv + head * HD + c);
    } else {
      kx[s] = vx[s] = make_uint4(0, 0, 0, 0);
    }
  }
  __shared__ float s_max[2][THREADS / 32];
  __shared__ unsigned s_nan[2];  // bit r: row r holds a NaN in its key or value
  if (threadIdx.x < 2) s_nan[threadIdx.x] = 0;
  __syncthreads();
  // Magnitudes as bf16 bit patterns (they order as integers), two to a word; inf and NaN are at or above 0x7f80.
  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    mk = max_u16x2(mk, largest(kx[s]));
    mv = max_u16x2(mv, largest(vx[s]));
  }
  mk = max(mk & 0xffffu, mk >> 16);
  mv = max(mv & 0xffffu, mv >> 16);
  if (max(mk, mv) >= 0x7f80u) {  // element by element: the largest finite one, and the rows with a NaN
    mk = mv = 0;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const bool nan_k = finite_max(kx[s], mk), nan_v = finite_max(vx[s], mv);
      const int r = (s * THREADS + (int)threadIdx.x) / VEC;
      if (nan_k || nan_v) atomicOr(&s_nan[r / 32], 1u << (r & 31));
    }
  }
  mk = __reduce_max_sync(0xffffffffu, mk);
  mv = __reduce_max_sync(0xffffffffu, mv);
  if (lane == 0) {
    s_max[0][warp] = __uint_as_float(mk << 16);
    s_max[1][warp] = __uint_as_float(mv << 16);
  }
  __syncthreads();
  float ak = 0.f, av = 0.f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    ak = fmaxf(ak, s_max[0][w]);
    av = fmaxf(av, s_max[1][w]);
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* scale = which ? a.v_scale : a.k_scale;
    uint8_t* codes = (which ? a.v_codes : a.k_codes) + at * BLOCK * HD;
    int e = scale_exponent(which ? av : ak);
    if (off > 0) {
      const int old = min(max((int)((__float_as_uint(old_scale[which]) >> 23) & 255u) - 127, E_MIN), E_MAX);
      if (e > old) {
        const float f = power_of_two(max(old - e, -126));
        for (int p = threadIdx.x; p < off * HD / 4; p += THREADS) {
          uint32_t w = reinterpret_cast<uint32_t*>(codes)[p];
          const float2 x = from_e4m3x2(w), y = from_e4m3x2(w >> 16);
          reinterpret_cast<uint32_t*>(codes)[p] = e4m3x2(x.x * f, x.y * f) | (e4m3x2(y.x * f, y.y * f) << 16);
        }
      } else {
        e = old;
      }
    }
    if (threadIdx.x == 0) scale[at] = power_of_two(e);
    const float inv = power_of_two(-e);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int p = s * THREADS + threadIdx.x, r = p / VEC, c = (p % VEC) * 8;
      if (r >= live) continue;
      const uint4 x4 = which ? vx[s] : kx[s];
      const uint32_t w[4] = {x4.x, x4.y, x4.z, x4.w};
      uint32_t o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 x = __fmul2_rn(unpack_bf16x2(w[q]), make_float2(inv, inv));
        o[q] = e4m3x2(x.x, x.y);
      }
      uint2 out = make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
      // A token with a NaN anywhere is a NaN key and a zero value: its scores are NaN wherever it is seen and its
      // value harms no row that does not see it (a masked probability of 0 times NaN would).
      if ((s_nan[r / 32] >> (r & 31)) & 1u)
        out = which ? make_uint2(0, 0) : make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
      *reinterpret_cast<uint2*>(codes + (int64_t)(off + r) * HD + c) = out;
    }
  }
}

// The kernel's limit on shared memory, raised once a device to what the most requests of the largest pool need: a limit
// set call by call could fall between another thread's check and its launch, and 48 KB without one count the static
// arrays too.
static int table_smem(int most_ints, const void* kernel, bool (&configured)[64], const char* what) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(KD_ERR_ARGUMENT, "kv tables: device index");
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most_ints * 4);
    if (e != cudaSuccess) return record_cuda_error(e, what);
    configured[dev] = true;
  }
  return KD_OK;
}
constexpr int assign_ints(int n, int capacity) { return 3 * n + 1 + seen_words(capacity); }
constexpr int release_ints(int n, int capacity) { return 2 * n + seen_words(capacity); }
static_assert(assign_ints(MAX_REQUESTS, 0x7fffffff) * 4 + 1024 <= 227 * 1024, "shared memory budget");

}  // namespace kv
}  // namespace kd

using namespace kd;

extern "C" int kd_kv_assign(const int32_t* lens, const int32_t* cu, int num_requests, int64_t rows, int32_t* table,
                            int64_t ld_table, int table_width, const int32_t* free_blocks, int capacity,
                            int32_t* free_count, int32_t* kv_len, int64_t* seqpos, int64_t* slots,
                            cudaStream_t stream) {
  if (num_requests < 0 || num_requests > kv::MAX_REQUESTS || rows < 0 || rows > 0x7fffffff || capacity < 0 ||
      table_width < 0 || ld_table < table_width)
    return set_error(KD_ERR_ARGUMENT, "kv_assign: 0 to 16384 requests, rows below 2^31, a table of its own width");
  if (!free_count || !cu || (num_requests && (!lens || !table || !kv_len)) || (rows && (!seqpos || !slots)) ||
      (capacity && !free_blocks))
    return set_error(KD_ERR_ARGUMENT, "kv_assign: null pointer");
  const kv::AssignArgs a{lens, cu, num_requests, rows, table, ld_table, table_width, free_blocks, capacity, free_count,
                         kv_len, seqpos, slots};
  static bool configured[64] = {false};
  if (int rc = kv::table_smem(kv::assign_ints(kv::MAX_REQUESTS, 0x7fffffff), (const void*)kv::assign_kernel, configured,
                              "kv_assign: shared memory"))
    return rc;
  int ctas = 1;  // a cluster's worth of rows: 1,024 rows a CTA and pass
  while (ctas < 8 && rows > (int64_t)ctas * kv::TABLE_THREADS) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kv::TABLE_THREADS);
  cfg.dynamicSmemBytes = kv::assign_ints(num_requests, capacity) * 4;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return record_cuda_error(cudaLaunchKernelEx(&cfg, kv::assign_kernel, a), "kv_assign: launch");
}

extern "C" int kd_kv_release(int32_t* table, int64_t ld_table, int table_width, const int32_t* lens,
                             const int32_t* keep, int num_requests, int32_t* free_blocks, int capacity,
                             int32_t* free_count, cudaStream_t stream) {
  if (num_requests < 0 || num_requests > kv::MAX_REQUESTS || capacity < 0 || table_width < 0 || ld_table < table_width)
    return set_error(KD_ERR_ARGUMENT, "kv_release: 0 to 16384 requests, a table of its own width");
  if (num_requests == 0) return KD_OK;
  if (!table || !lens || !keep || !free_blocks || !free_count)
    return set_error(KD_ERR_ARGUMENT, "kv_release: null pointer");
  const kv::ReleaseArgs a{table, ld_table, table_width, lens, keep, num_requests, free_blocks, capacity, free_count};
  static bool configured[64] = {false};
  if (int rc = kv::table_smem(kv::release_ints(kv::MAX_REQUESTS, 0x7fffffff), (const void*)kv::release_kernel,
                              configured, "kv_release: shared memory"))
    return rc;
  kv::release_kernel<<<1, kv::TABLE_THREADS, kv::release_ints(num_requests, capacity) * 4, stream>>>(a);
  return record_cuda_error(cudaGetLastError(), "kv_release: launch");
}

extern "C" int kd_kv_store_e4m3(const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t rows,
                                const int32_t* cu, int num_requests, const int64_t* slots, int num_heads_kv,
                                int head_dim, void* k_codes, void* v_codes, float* k_scale, float* v_scale,
                                int64_t num_blocks, cudaStream_t stream) {
  if (num_requests < 0 || num_requests > kv::MAX_REQUESTS || rows < 0 || rows > 0x7fffffff || num_blocks < 0 ||
      num_blocks > 0x7fffffff)
    return set_error(KD_ERR_ARGUMENT, "kv_store: 0 to 16384 requests, rows and blocks below 2^31");
  if (num_heads_kv <= 0 || num_heads_kv > 65535)
    return set_error(KD_ERR_ARGUMENT, "kv_store: 1 to 65535 key/value heads");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512)
    return set_error(KD_ERR_ARGUMENT, "kv_store: head_dim must be 64, 128, 256 or 512");
  if (num_requests == 0 || rows == 0 || num_blocks == 0) return KD_OK;
  if (!k || !v || !cu || !slots || !k_codes || !v_codes || !k_scale || !v_scale)
    return set_error(KD_ERR_ARGUMENT, "kv_store: null pointer");
  auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (!a16(k) || !a16(v) || !a16(k_codes) || !a16(v_codes) || ldk % 8 || ldv % 8)
    return set_error(KD_ERR_ARGUMENT, "kv_store: pointers and row strides must be 16-byte aligned");
  if (ldk < (int64_t)num_heads_kv * head_dim || ldv < (int64_t)num_heads_kv * head_dim)
    return set_error(KD_ERR_ARGUMENT, "kv_store: row strides smaller than heads x head_dim");
  const kv::StoreArgs a{static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v), ldk, ldv, rows, cu,
                        num_requests, num_heads_kv, slots, num_blocks, static_cast<uint8_t*>(k_codes),
                        static_cast<uint8_t*>(v_codes), k_scale, v_scale};
  const dim3 grid((unsigned)(rows / kv::BLOCK + 2 * (int64_t)num_requests), num_heads_kv);
  switch (head_dim) {
    case 64:
      kv::store_kernel<64><<<grid, kv::store_threads(64), 0, stream>>>(a);
      break;
    case 128:
      kv::store_kernel<128><<<grid, kv::store_threads(128), 0, stream>>>(a);
      break;
    case 256:
      kv::store_kernel<256><<<grid, kv::store_threads(256), 0, stream>>>(a);
      break;
    default:
      kv::store_kernel<512><<<grid, kv::store_threads(512), 0, stream>>>(a);
  }
  return record_cuda_error(cudaGetLastError(), "kv_store: launch");
}
