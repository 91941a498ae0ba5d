// What the two kernels of the attention over cached blocks share: arguments, a request's geometry, exact conversions of
// e4m3 codes and powers of two.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "kd_internal.h"

namespace kd {
namespace ca {

constexpr int BN = KD_KV_BLOCK;  // keys per tile: one block

struct Args {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const __nv_bfloat16* gate;
  int64_t ldq, ldo, ldg;
  const int32_t* table;
  int64_t ldt;
  int width;
  const int32_t* cu;
  const int32_t* kv_len;
  int n;
  int64_t total_q;
  const float* k_scale;
  const float* v_scale;
  int blocks;
  int hq, hkv, group;
  float scale_log2;
  int left, right;
  int* items;   // scratch of the kernel for few rows: the number of items
  void* descs;  // what the joining launch needs of an item (few rows), or of one that several CTAs share (many)
  float* partials;
  int* status;
};

struct Request {
  int q0, lq, lk;
  int first, tiles;  // key tiles that any row may see
};

KD_DEVICE Request request(const Args& a, int i) {
  Request r;
  r.q0 = a.cu[i];
  const int end = a.cu[i + 1];
  r.lq = r.q0 < 0 || end > a.total_q ? 0 : max(end - r.q0, 0);
  r.lk = (int)min((int64_t)max(a.kv_len[i], 0), (int64_t)a.width * BN);
  const int kmin = a.left >= 0 ? max(0, r.lk - r.lq - a.left) : 0;
  r.first = kmin / BN;
  r.tiles = r.lq > 0 && r.lk > kmin ? (r.lk - 1) / BN - r.first + 1 : 0;
  return r;
}

// Quotients of non-negative numbers: in 32 bits where both fit (a 64-bit division costs some 600 cycles here, and the
// first key tile waits for several).
KD_DEVICE int64_t quotient(int64_t a, int64_t b) {
  return ((uint64_t)a | (uint64_t)b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// CTAs that take part: every one of them has a tile, so no partial of an item is missing.
KD_DEVICE int64_t shares(int64_t total, int ctas) { return total < ctas ? (total > 0 ? total : 1) : ctas; }

KD_DEVICE float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^e for whole e, clamped to the normal float32 exponents.
KD_DEVICE float pow2i(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }
// The exponent of a scale (a power of two).
KD_DEVICE int exponent_of(float s) { return (int)((__float_as_uint(s) >> 23) & 255u) - 127; }

// Four e4m3 codes to two f16 pairs (exact).
KD_DEVICE void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

// Two values as packed e4m3 codes, round to nearest even, saturating at +-448; NaN stays NaN.
KD_DEVICE uint32_t e4m3_pair(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// The softmax scale * log2(e) * a query row's power of two (`row`), times a block's key scale: finite and not 0, so that
// it times a masked -inf or a score of 0 is no NaN.
KD_DEVICE float score_factor(float row, float k_scale) {
  return fminf(fmaxf(row * k_scale, 1.1754944e-38f), 3.4028235e38f);
}

KD_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// A warpgroup's share of the block's registers (executed by all of it, one instruction).
template <int N>
KD_DEVICE void set_registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
KD_DEVICE void set_registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Launches the joining kernel so that its blocks are in place when the kernel before it in the stream ends (it waits for
// that itself, by griddepcontrol.wait).
template <typename K>
int launch_after(K kernel, dim3 grid, int threads, cudaStream_t stream, const Args& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return record_cuda_error(cudaLaunchKernelEx(&cfg, kernel, a), "attention_cache: join launch");
}

// The kernel for many rows per key/value head (cache_attention_tiles.cu).
int64_t row_tiles_workspace(int head_dim, int sms);
int row_tiles(int head_dim, const Args& a, const void* k_codes, const void* v_codes, uint8_t* ws, int64_t ws_bytes,
              cudaStream_t stream);

}  // namespace ca
}  // namespace kd
