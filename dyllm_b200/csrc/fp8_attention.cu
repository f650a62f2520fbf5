// Exact attention of listed query rows over 8-bit keys and values (fp8_cache.cuh), in place in their caches:
//
//   s_j = scale * (q . k_j);   s_j = cap * tanh(s_j / cap)  (cap > 0);   s_j -= slope_h * |pos_q - pos_j|
//   o   = sum_j softmax(s)_j v_j     over the visible keys of the row's sequence; no visible key: o = 0
//
// A value is code * 2^e(j).  With t_j = s_j * log2(e) the weights are taken as
//   w_j = 2^(t_j + e(j) - m'),  m' = max_j (t_j + e(j)),   o = sum_j w_j code_j / sum_j w_j 2^-e(j),
// which needs one exponential per score, and w <= 1 whatever the scales are: a weight that vanishes next to the largest one
// belongs to a value that vanishes next to the largest.
#include "fp8_cache.cuh"

namespace dyllm {
namespace {

constexpr int kD = 128;
constexpr float kLog2e = 1.4426950408889634f;

struct Fp8AttnParams {
  const __nv_bfloat16* q;
  int64_t ldq;
  int total_q;
  const uint8_t* k_codes;
  const float* k_scales;
  int64_t k_rows;
  const uint8_t* v_codes;
  const float* v_scales;
  int64_t v_rows;
  const int64_t* k_starts;
  const int64_t* v_starts;
  const int64_t* seq_ids;
  __nv_bfloat16* out;
  const int32_t* cu_q;
  const int32_t* cu_k;
  const int32_t* cu_sal;
  const int32_t* idx;
  int num_salient, batch, H, Hkv;
  float scale, cap;
  const float* slopes;
  const int2* ranges;
};

// First rows of sequence b in the two caches and the number of its keys that lie in both (0: a sequence without a cache).
struct KeyRange {
  int64_t k0, v0;
  int len;
};
__device__ __forceinline__ KeyRange keys_of(const Fp8AttnParams& p, int b) {
  KeyRange r;
  const int64_t sid = __ldg(p.seq_ids + b);
  r.k0 = __ldg(p.k_starts + sid);
  r.v0 = __ldg(p.v_starts + sid);
  int64_t len = __ldg(p.cu_k + b + 1) - __ldg(p.cu_k + b);
  len = min(len, min(p.k_rows - r.k0, p.v_rows - r.v0));
  r.len = r.k0 < 0 || r.v0 < 0 || len < 0 ? 0 : static_cast<int>(len);
  return r;
}

// t = s * log2(e) of one score from the product of the codes.
__device__ __forceinline__ float score_log2(float dot_scaled, float cap, float inv_cap, float slope, int distance) {
  float s = dot_scaled;
  if (cap > 0.f) {
    // tanh(x) = 1 - 2 / (1 + e^2x): an absolute error of a few 2^-24 (the hardware tanh has 2^-11)
    s = cap - 2.f * cap * __frcp_rn(1.f + exp2f(2.f * kLog2e * inv_cap * s));
  }
  return (s - slope * static_cast<float>(distance)) * kLog2e;
}

__device__ __forceinline__ float value_exponent(float scale) {
  const uint32_t bits = __float_as_uint(scale);
  if (bits >= 0x7f800000u)
    return __uint_as_float(0x7fc00000u);
  return static_cast<float>(max(static_cast<int>(bits >> 23) - 127, kFp8MinExp));
}

// One warp per (listed row, head), 32 keys at a time: lane j keeps the score of key j, a lane holds four head dimensions.
__global__ void __launch_bounds__(256) fp8_rows_simple_kernel(const Fp8AttnParams p) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int group = p.H / p.Hkv;
  const int n = min(p.num_salient, __ldg(p.cu_sal + p.batch));
  const int64_t total = static_cast<int64_t>(n) * p.H;
  for (int64_t w = blockIdx.x * 8ll + (threadIdx.x >> 5); w < total; w += gridDim.x * 8ll) {
    const int i = static_cast<int>(w / p.H), h = static_cast<int>(w - static_cast<int64_t>(i) * p.H), hk = h / group;
    int b = 0;
    while (b < p.batch - 1 && __ldg(p.cu_sal + b + 1) <= i)
      ++b;
    const int r = __ldg(p.idx + i);
    const KeyRange kr = keys_of(p, b);
    const int pos = __ldg(p.cu_k + b + 1) - __ldg(p.cu_k + b) - (__ldg(p.cu_q + b + 1) - r);
    int lo = 0, hi = kr.len;
    float q[4] = {0.f, 0.f, 0.f, 0.f};
    if (r >= 0 && r < p.total_q) {
      const __nv_bfloat162* src = reinterpret_cast<const __nv_bfloat162*>(p.q + r * p.ldq + h * kD) + lane * 2;
      const float2 a = __bfloat1622float2(src[0]), c = __bfloat1622float2(src[1]);
      q[0] = a.x, q[1] = a.y, q[2] = c.x, q[3] = c.y;
      if (p.ranges) {
        const int2 v = __ldg(p.ranges + r);
        lo = max(lo, v.x);
        hi = min(hi, v.y);
      }
    } else {
      hi = 0;
    }
    const float slope = p.slopes ? __ldg(p.slopes + h) : 0.f;
    const float inv_cap = p.cap > 0.f ? 1.f / p.cap : 0.f;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int base = lo; base < hi; base += 32) {
      const int live = min(32, hi - base);
      float dot = 0.f;
      for (int j = 0; j < live; ++j) {
        const uint32_t c = *reinterpret_cast<const uint32_t*>(p.k_codes + ((kr.k0 + base + j) * p.Hkv + hk) * kD + lane * 4);
        const float2 a = fp8_to_float2(c & 0xffffu), d = fp8_to_float2(c >> 16);
        float x = q[0] * a.x + q[1] * a.y + q[2] * d.x + q[3] * d.y;
#pragma unroll
        for (int s = 16; s; s >>= 1)
          x += __shfl_xor_sync(0xffffffffu, x, s);
        dot = lane == j ? x : dot;
      }
      float t = -INFINITY, inv = 0.f;
      if (lane < live) {
        const int j = base + lane;
        const float e = value_exponent(__ldg(p.v_scales + (kr.v0 + j) * p.Hkv + hk));
        inv = exp2f(-e);
        t = score_log2(dot * __ldg(p.k_scales + (kr.k0 + j) * p.Hkv + hk) * p.scale, p.cap, inv_cap, slope, abs(pos - j)) + e;
      }
      float top = t;
#pragma unroll
      for (int s = 16; s; s >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
      const float now = fmaxf(m, top);
      const float base_m = now == -INFINITY ? 0.f : now;
      const float old = exp2f(m - base_m);
      const float wt = lane < live ? exp2f(t - base_m) : 0.f;
      m = now;
      l = l * old + wt * inv;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        o[d] *= old;
      for (int j = 0; j < live; ++j) {
        const float wj = __shfl_sync(0xffffffffu, wt, j);
        const uint32_t c = *reinterpret_cast<const uint32_t*>(p.v_codes + ((kr.v0 + base + j) * p.Hkv + hk) * kD + lane * 4);
        const float2 a = fp8_to_float2(c & 0xffffu), d = fp8_to_float2(c >> 16);
        o[0] += wj * a.x, o[1] += wj * a.y, o[2] += wj * d.x, o[3] += wj * d.y;
      }
    }
#pragma unroll
    for (int s = 16; s; s >>= 1)
      l += __shfl_xor_sync(0xffffffffu, l, s);
    const float inv_l = lo < hi ? 1.f / l : 0.f;
    __nv_bfloat162* dst = reinterpret_cast<__nv_bfloat162*>(p.out + (static_cast<int64_t>(i) * p.H + h) * kD) + lane * 2;
    dst[0] = __floats2bfloat162_rn(o[0] * inv_l, o[1] * inv_l);
    dst[1] = __floats2bfloat162_rn(o[2] * inv_l, o[3] * inv_l);
  }
}

}  // namespace
}  // namespace dyllm

using namespace dyllm;

extern "C" {

size_t dyllm_attention_salient_rows_fp8_workspace_bytes(int num_salient, int batch, int num_heads, int num_kv_heads) {
  return 0;
}

int dyllm_attention_salient_rows_fp8(const void* q, int64_t ldq, int total_q, const void* k_codes, const float* k_scales,
                                     int64_t k_rows, const void* v_codes, const float* v_scales, int64_t v_rows,
                                     const int64_t* k_seq_starts, const int64_t* v_seq_starts, const int64_t* seq_ids,
                                     void* out, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                                     int max_rows_per_seq, int num_heads, int num_kv_heads, int head_dim,
                                     const int32_t* cu_salientlens, const int32_t* idx_salient_row, int num_salient,
                                     float scale, float softcap, const float* slopes, const int32_t* key_ranges,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  DYLLM_REQUIRE(head_dim == kD, DYLLM_ERR_UNSUPPORTED, "attention_salient_rows_fp8: head_dim %d (only 128 is built)", head_dim);
  DYLLM_REQUIRE(batch >= 0 && total_q >= 0 && num_salient >= 0 && max_rows_per_seq >= 0 && k_rows >= 0 && v_rows >= 0,
                DYLLM_ERR_INVALID_ARGUMENT, "attention_salient_rows_fp8: batch %d Tq %d rows %d max rows %d", batch, total_q,
                num_salient, max_rows_per_seq);
  DYLLM_REQUIRE(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0, DYLLM_ERR_INVALID_ARGUMENT,
                "attention_salient_rows_fp8: query heads (%d) must be a positive multiple of KV heads (%d)", num_heads,
                num_kv_heads);
  DYLLM_REQUIRE(scale == scale && softcap >= 0.f && softcap <= 3.0e38f, DYLLM_ERR_INVALID_ARGUMENT,
                "attention_salient_rows_fp8: scale %g softcap %g", static_cast<double>(scale), static_cast<double>(softcap));
  if (batch == 0 || num_salient == 0 || max_rows_per_seq == 0)
    return DYLLM_OK;
  DYLLM_REQUIRE(q && k_codes && k_scales && v_codes && v_scales && k_seq_starts && v_seq_starts && seq_ids && out &&
                    cu_seqlens_q && cu_seqlens_k && cu_salientlens && idx_salient_row,
                DYLLM_ERR_INVALID_ARGUMENT, "attention_salient_rows_fp8: null pointer");
  for (const void* p16 : {q, k_codes, v_codes, static_cast<const void*>(out)})
    DYLLM_REQUIRE((reinterpret_cast<uintptr_t>(p16) & 15) == 0, DYLLM_ERR_INVALID_ARGUMENT,
                  "attention_salient_rows_fp8: q, codes and out must be 16-byte aligned");
  DYLLM_REQUIRE(ldq % 8 == 0 && ldq >= static_cast<int64_t>(num_heads) * kD, DYLLM_ERR_INVALID_ARGUMENT,
                "attention_salient_rows_fp8: the row pitch of q (%lld) must be a multiple of 8 and at least heads * 128",
                static_cast<long long>(ldq));
  DYLLM_REQUIRE((reinterpret_cast<uintptr_t>(key_ranges) & 7) == 0, DYLLM_ERR_INVALID_ARGUMENT,
                "attention_salient_rows_fp8: key_ranges must be 8-byte aligned");
  Fp8AttnParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.ldq = ldq;
  p.total_q = total_q;
  p.k_codes = static_cast<const uint8_t*>(k_codes);
  p.k_scales = k_scales;
  p.k_rows = k_rows;
  p.v_codes = static_cast<const uint8_t*>(v_codes);
  p.v_scales = v_scales;
  p.v_rows = v_rows;
  p.k_starts = k_seq_starts;
  p.v_starts = v_seq_starts;
  p.seq_ids = seq_ids;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.cu_sal = cu_salientlens;
  p.idx = idx_salient_row;
  p.num_salient = num_salient;
  p.batch = batch;
  p.H = num_heads;
  p.Hkv = num_kv_heads;
  p.scale = scale;
  p.cap = softcap;
  p.slopes = slopes;
  p.ranges = reinterpret_cast<const int2*>(key_ranges);
  const int64_t want = (static_cast<int64_t>(num_salient) * num_heads + 7) / 8, cap = sm_count() * 8ll;
  DYLLM_LAUNCH(fp8_rows_simple_kernel, static_cast<unsigned>(want < cap ? want : cap), 256, 0,
               static_cast<cudaStream_t>(stream), p);
  return check_launch("attention_salient_rows_fp8");
}

}  // extern "C"
