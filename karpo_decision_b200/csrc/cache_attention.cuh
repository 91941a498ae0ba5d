// What the two kernels of the attention over cached blocks share: arguments, a request's geometry, exact conversions of
// e4m3 codes and powers of two.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "kd_internal.h"

namespace kd {
namespace ca {

constexpr int BN = KD_KV_BLOCK;  // keys per tile: one block
constexpr int RT = 16;           // query rows per tile of the kernel for few rows

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
  int64_t* tile_cu;   // [n + 1] few rows: key tiles of the requests before (of one key/value head); many: their weights
  int32_t* item_cu;   // [n + 1] few rows: 16-row tiles of the requests before
  float* partials;
  int* status;
};

struct Request {
  int q0, lq, lk;
  int nrt;          // 16-row tiles
  int first, tiles; // key tiles that any row may see
};

KD_DEVICE Request request(const Args& a, int i) {
  Request r;
  r.q0 = a.cu[i];
  const int end = a.cu[i + 1];
  r.lq = r.q0 < 0 || end > a.total_q ? 0 : max(end - r.q0, 0);
  r.lk = (int)min((int64_t)max(a.kv_len[i], 0), (int64_t)a.width * BN);
  r.nrt = (int)(((int64_t)r.lq * a.group + RT - 1) / RT);
  const int kmin = a.left >= 0 ? max(0, r.lk - r.lq - a.left) : 0;
  r.first = kmin / BN;
  r.tiles = r.lq > 0 && r.lk > kmin ? (r.lk - 1) / BN - r.first + 1 : 0;
  return r;
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

// scale * log2(e) times the power-of-two scales of a query row and a block's keys: finite and not 0, so that it times a
// masked -inf or a score of 0 is no NaN.
KD_DEVICE float score_factor(float q_scale, float k_scale, float scale_log2) {
  return fminf(fmaxf(q_scale * k_scale * scale_log2, 1.1754944e-38f), 3.4028235e38f);
}

KD_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The kernel for many rows per key/value head (cache_attention_tiles.cu).
int64_t row_tiles_workspace(int head_dim, int n, int sms);
int row_tiles(int head_dim, const Args& a, const void* k_codes, const void* v_codes, uint8_t* ws, int64_t ws_bytes,
              cudaStream_t stream);

}  // namespace ca
}  // namespace kd
