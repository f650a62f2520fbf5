// 8-bit caches of keys and values: quantised as they are written, read back as bf16 (fp8_cache.cuh has the format).
//
// All three kernels give a warp one row and up to 4 G of its heads, eight threads to a head: thread p holds the values 8p .. 8p+7
// and 64+8p .. 64+8p+7 (the two halves that the rotary embedding pairs), so the 16-byte loads of the eight are contiguous, the
// amax is three shuffles and the codes leave as 8-byte stores of 64 contiguous bytes.  HBM-bound: 388 bytes per (row, head) for
// write and read.  All loads of a warp are in flight at once, beside the search for its sequence.
#include <type_traits>

#include "fp8_cache.cuh"

namespace dyllm {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;

// Number of sequences that end at or before a row (cu ascends); for a whole warp, 32 places at a time.
__device__ __forceinline__ int seq_of_row(const int32_t* __restrict__ cu, int batch, int64_t row) {
  int lo = 0;
  for (int n = batch;;) {
    const int step = (n + 31) >> 5, k = lo + (static_cast<int>(lane_id()) + 1) * step;
    const bool ends = k <= lo + n && static_cast<int64_t>(__ldg(cu + k)) <= row;
    lo += __popc(__ballot_sync(0xffffffffu, ends)) * step;
    if (step <= 1)
      return lo;
    n = min(step, batch - lo);
  }
}

// Cache row of packed row p: its sequence's first row + its place, or (cu_k given) its place among the sequence's last rows.
// -1: no such row in the cache; -2: the row belongs to no sequence.
__device__ __forceinline__ int64_t cache_row_of(int p, const int64_t* __restrict__ seq_starts,
                                                const int32_t* __restrict__ cu, const int32_t* __restrict__ cu_k,
                                                const int64_t* __restrict__ seq_ids, int batch, int64_t cache_rows) {
  const int b = seq_of_row(cu, batch, p);
  if (b >= batch)
    return -2;
  const int first = __ldg(cu + b);
  if (p < first)
    return -2;
  const int64_t start = __ldg(seq_starts + __ldg(seq_ids + b));
  int64_t row = start + (p - first);
  if (cu_k)
    row += (__ldg(cu_k + b + 1) - __ldg(cu_k + b)) - (__ldg(cu + b + 1) - first);
  return start < 0 || row < start || row >= cache_rows ? -1 : row;
}

template <int G>
__global__ void __launch_bounds__(kThreads)
fp8_cache_write_kernel(const uint4* __restrict__ x, int64_t ldx, int heads, uint2* __restrict__ codes,
                       float* __restrict__ scales, int64_t cache_rows, const int64_t* __restrict__ seq_starts,
                       const int32_t* __restrict__ cu, const int32_t* __restrict__ cu_k,
                       const int64_t* __restrict__ seq_ids, int batch, int rows) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  const int p = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = lane_id(), part = lane & 7;
  const int h0 = blockIdx.y * 4 * G + (lane >> 3);
  if (p >= rows)
    return;
  const uint4* src = x + p * ldx + h0 * 16 + part;
  uint4 a[G], b[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    a[g] = b[g] = make_uint4(0u, 0u, 0u, 0u);
    if (h0 + 4 * g < heads) {
      a[g] = __ldcs(src + g * 64);
      b[g] = __ldcs(src + g * 64 + 8);
    }
  }
  const int64_t row = cache_row_of(p, seq_starts, cu, cu_k, seq_ids, batch, cache_rows);
  if (row < 0)
    return;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float v[16];
    bf16x8_to_float(a[g], v);
    bf16x8_to_float(b[g], v + 8);
    uint2 lo, hi;
    const uint32_t scale = fp8_quantise16(v, lo, hi);
    if (h0 + 4 * g < heads) {
      const int64_t at = row * heads + h0 + 4 * g;
      codes[at * 16 + part] = lo;
      codes[at * 16 + part + 8] = hi;
      if (part == 0)
        scales[at] = __uint_as_float(scale);
    }
  }
}

template <int G>
__global__ void __launch_bounds__(kThreads)
fp8_cache_read_kernel(const uint2* __restrict__ codes, const float* __restrict__ scales, int64_t cache_rows, int heads,
                      uint4* __restrict__ out, const int64_t* __restrict__ seq_starts, const int32_t* __restrict__ cu,
                      const int32_t* __restrict__ cu_k, const int64_t* __restrict__ seq_ids, int batch, int rows) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  const int p = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = lane_id(), part = lane & 7;
  const int h0 = blockIdx.y * 4 * G + (lane >> 3);
  if (p >= rows)
    return;
  const int64_t row = cache_row_of(p, seq_starts, cu, cu_k, seq_ids, batch, cache_rows);
  if (row == -2)
    return;
  uint2 lo[G], hi[G];
  float scale[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    lo[g] = hi[g] = make_uint2(0u, 0u);
    scale[g] = 0.f;
    if (row >= 0 && h0 + 4 * g < heads) {
      const int64_t at = row * heads + h0 + 4 * g;
      lo[g] = __ldg(codes + at * 16 + part);
      hi[g] = __ldg(codes + at * 16 + part + 8);
      scale[g] = __ldg(scales + at);
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (h0 + 4 * g < heads) {
      float v[16];
      fp8x8_to_float(lo[g], scale[g], v);
      fp8x8_to_float(hi[g], scale[g], v + 8);
      uint4* dst = out + (static_cast<int64_t>(p) * heads + h0 + 4 * g) * 16 + part;
      __stcs(dst, float_to_bf16x8(v));
      __stcs(dst + 8, float_to_bf16x8(v + 8));
    }
}

// The products and sums of the rotation are rounded one by one (no fused multiply-add), so that the codes are those of the
// same rotation written with separate operations.
template <int G>
__global__ void __launch_bounds__(kThreads)
fp8_kv_cache_update_kernel(const uint4* __restrict__ k_new, int64_t ldk, const uint4* __restrict__ v_new, int64_t ldv,
                           const int64_t* __restrict__ rows_k, const int64_t* __restrict__ positions,
                           const int64_t* __restrict__ pos_idx, const float4* __restrict__ cos_sin, int max_pos,
                           const int32_t* __restrict__ cu_k, const int64_t* __restrict__ k_starts,
                           const int64_t* __restrict__ v_starts, const int64_t* __restrict__ seq_ids, int batch,
                           int num_rows, const int32_t* __restrict__ num_rows_dev, int heads, uint2* k_codes,
                           float* k_scales, int64_t k_rows, uint2* v_codes, float* v_scales, int64_t v_rows,
                           uint4* __restrict__ dv) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  const int i = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = lane_id(), part = lane & 7;
  const int h0 = blockIdx.y * 4 * G + (lane >> 3);
  if (i >= (num_rows_dev ? min(num_rows, __ldg(num_rows_dev)) : num_rows))
    return;
  const uint4* ksrc = k_new + i * ldk + h0 * 16 + part;
  const uint4* vsrc = v_new + i * ldv + h0 * 16 + part;
  uint4 ka[G], kb[G], va[G], vb[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    ka[g] = kb[g] = va[g] = vb[g] = make_uint4(0u, 0u, 0u, 0u);
    if (h0 + 4 * g < heads) {
      ka[g] = __ldcs(ksrc + g * 64);
      kb[g] = __ldcs(ksrc + g * 64 + 8);
      va[g] = __ldcs(vsrc + g * 64);
      vb[g] = __ldcs(vsrc + g * 64 + 8);
    }
  }
  int64_t pos = __ldg(positions + (pos_idx ? __ldg(pos_idx + i) : i));
  pos = pos < 0 ? 0 : (pos >= max_pos ? max_pos - 1 : pos);
  const float4* cs = cos_sin + pos * 32 + part * 2;
  float c[8], s[8];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    *reinterpret_cast<float4*>(c + 4 * j) = __ldg(cs + j);
    *reinterpret_cast<float4*>(s + 4 * j) = __ldg(cs + 16 + j);
  }
  const int64_t r = __ldg(rows_k + i);
  const int b = min(seq_of_row(cu_k, batch, r), batch - 1);
  const int32_t first = __ldg(cu_k + b);
  const int64_t off = r - first, length = __ldg(cu_k + b + 1) - first, sid = __ldg(seq_ids + b);
  const int64_t krow = __ldg(k_starts + sid) + off, vrow = __ldg(v_starts + sid) + off;
  // a row that no cache holds (a sequence without one, an index out of range) changes nothing: its delta-V is zero.  Behind the
  // batch's last row the caches may go on, with sequences of others.
  const bool held = off >= 0 && off < length && krow >= off && krow < k_rows && vrow >= off && vrow < v_rows;
  uint2 olo[G], ohi[G];
  float oscale[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    olo[g] = ohi[g] = make_uint2(0u, 0u);
    oscale[g] = 0.f;
    if (held && h0 + 4 * g < heads) {
      const int64_t at = vrow * heads + h0 + 4 * g;
      olo[g] = v_codes[at * 16 + part];
      ohi[g] = v_codes[at * 16 + part + 8];
      oscale[g] = v_scales[at];
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const bool head = h0 + 4 * g < heads, store = held && head;
    float x[16], y[16];
    uint2 lo, hi;
    bf16x8_to_float(ka[g], y);
    bf16x8_to_float(kb[g], y + 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = __fsub_rn(__fmul_rn(y[j], c[j]), __fmul_rn(y[8 + j], s[j]));
      x[8 + j] = __fadd_rn(__fmul_rn(y[8 + j], c[j]), __fmul_rn(y[j], s[j]));
    }
    const uint32_t kscale = fp8_quantise16(x, lo, hi);
    if (store) {
      const int64_t at = krow * heads + h0 + 4 * g;
      k_codes[at * 16 + part] = lo;
      k_codes[at * 16 + part + 8] = hi;
      if (part == 0)
        k_scales[at] = __uint_as_float(kscale);
    }
    bf16x8_to_float(va[g], x);
    bf16x8_to_float(vb[g], x + 8);
    const uint32_t vscale = fp8_quantise16(x, lo, hi);
    fp8x8_to_float(lo, __uint_as_float(vscale), x);
    fp8x8_to_float(hi, __uint_as_float(vscale), x + 8);
    fp8x8_to_float(olo[g], oscale[g], y);
    fp8x8_to_float(ohi[g], oscale[g], y + 8);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      x[j] = held ? x[j] - y[j] : 0.f;
    if (store) {
      const int64_t at = vrow * heads + h0 + 4 * g;
      v_codes[at * 16 + part] = lo;
      v_codes[at * 16 + part + 8] = hi;
      if (part == 0)      // all eight threads have read the old one: the shuffles of the amax lie between
        v_scales[at] = __uint_as_float(vscale);
    }
    if (head) {
      uint4* dst = dv + (static_cast<int64_t>(i) * heads + h0 + 4 * g) * 16 + part;
      __stcs(dst, float_to_bf16x8(x));
      __stcs(dst + 8, float_to_bf16x8(x + 8));
    }
  }
}

template <int N>
using Groups = std::integral_constant<int, N>;

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Checks shared by the calls; 1 = there is work.
int check_heads(const char* name, int heads, int head_dim, int batch, int rows, int64_t cache_rows) {
  DYLLM_REQUIRE(head_dim == 128, DYLLM_ERR_UNSUPPORTED, "%s: head_dim %d (only 128 is built)", name, head_dim);
  DYLLM_REQUIRE(heads > 0 && batch >= 0 && rows >= 0 && cache_rows >= 0, DYLLM_ERR_INVALID_ARGUMENT,
                "%s: heads %d batch %d rows %d cache rows %lld", name, heads, batch, rows, static_cast<long long>(cache_rows));
  return rows > 0 && batch > 0 ? 1 : DYLLM_OK;
}

int check_stride(const char* name, const char* what, const void* x, int64_t ld, int heads) {
  DYLLM_REQUIRE(x, DYLLM_ERR_INVALID_ARGUMENT, "%s: null %s", name, what);
  DYLLM_REQUIRE(aligned(x, 16) && ld % 8 == 0 && ld >= static_cast<int64_t>(heads) * 128, DYLLM_ERR_INVALID_ARGUMENT,
                "%s: %s must be 16-byte aligned with a row pitch that is a multiple of 8 and at least heads * 128 (%lld)", name,
                what, static_cast<long long>(ld));
  return DYLLM_OK;
}

// One warp a row and 4 G heads; more heads a warp where there are enough rows to fill the GPU either way.
dim3 grid_of(int rows, int heads, int g) { return dim3((rows - 1) / kWarps + 1, (heads + 4 * g - 1) / (4 * g)); }
int groups_of(int rows, int heads, int most) {
  int g = most;
  while (g > 1 && (4 * (g / 2) >= heads || static_cast<int64_t>(rows) * heads < 64ll * g * sm_count()))
    g /= 2;
  return g;
}

}  // namespace
}  // namespace dyllm

using namespace dyllm;

extern "C" {

int dyllm_fp8_cache_write(const void* x, int64_t ldx, int heads, int head_dim, void* codes, float* scales,
                          int64_t cache_rows, const int64_t* seq_starts, const int32_t* cu_seqlens,
                          const int32_t* cu_seqlens_k, const int64_t* seq_ids, int batch, int total_rows, void* stream) {
  int rc = check_heads("fp8_cache_write", heads, head_dim, batch, total_rows, cache_rows);
  if (rc <= 0)
    return rc;
  if ((rc = check_stride("fp8_cache_write", "x", x, ldx, heads)) != DYLLM_OK)
    return rc;
  DYLLM_REQUIRE(((codes && scales) || cache_rows == 0) && seq_starts && cu_seqlens && seq_ids, DYLLM_ERR_INVALID_ARGUMENT,
                "fp8_cache_write: null pointer");
  DYLLM_REQUIRE(aligned(codes, 16) && aligned(scales, 4), DYLLM_ERR_INVALID_ARGUMENT,
                "fp8_cache_write: codes must be 16-byte aligned");
  auto launch = [&](auto groups) {
    constexpr int G = decltype(groups)::value;
    DYLLM_LAUNCH(fp8_cache_write_kernel<G>, grid_of(total_rows, heads, G), kThreads, 0, static_cast<cudaStream_t>(stream), static_cast<const uint4*>(x), ldx / 8, heads, static_cast<uint2*>(codes), scales, cache_rows, seq_starts, cu_seqlens, cu_seqlens_k, seq_ids, batch, total_rows);
  };
  const int g = groups_of(total_rows, heads, 4);
  g == 4 ? launch(Groups<4>()) : g == 2 ? launch(Groups<2>()) : launch(Groups<1>());
  return check_launch("fp8_cache_write");
}

int dyllm_fp8_cache_read(const void* codes, const float* scales, int64_t cache_rows, int heads, int head_dim, void* out,
                         const int64_t* seq_starts, const int32_t* cu_seqlens, const int32_t* cu_seqlens_k,
                         const int64_t* seq_ids, int batch, int total_rows, void* stream) {
  int rc = check_heads("fp8_cache_read", heads, head_dim, batch, total_rows, cache_rows);
  if (rc <= 0)
    return rc;
  DYLLM_REQUIRE(((codes && scales) || cache_rows == 0) && out && seq_starts && cu_seqlens && seq_ids, DYLLM_ERR_INVALID_ARGUMENT,
                "fp8_cache_read: null pointer");
  DYLLM_REQUIRE(aligned(codes, 16) && aligned(scales, 4) && aligned(out, 16), DYLLM_ERR_INVALID_ARGUMENT,
                "fp8_cache_read: codes and out must be 16-byte aligned");
  auto launch = [&](auto groups) {
    constexpr int G = decltype(groups)::value;
    DYLLM_LAUNCH(fp8_cache_read_kernel<G>, grid_of(total_rows, heads, G), kThreads, 0, static_cast<cudaStream_t>(stream), static_cast<const uint2*>(codes), scales, cache_rows, heads, static_cast<uint4*>(out), seq_starts, cu_seqlens, cu_seqlens_k, seq_ids, batch, total_rows);
  };
  const int g = groups_of(total_rows, heads, 4);
  g == 4 ? launch(Groups<4>()) : g == 2 ? launch(Groups<2>()) : launch(Groups<1>());
  return check_launch("fp8_cache_read");
}

int dyllm_fp8_kv_cache_update(const void* k_new, int64_t ldk, const void* v_new, int64_t ldv, const int64_t* rows_k,
                              const int64_t* positions, const int64_t* pos_idx, const float* cos_sin, int max_pos,
                              const int32_t* cu_seqlens_k, const int64_t* k_seq_starts, const int64_t* v_seq_starts,
                              const int64_t* seq_ids, int batch, int num_rows, const int32_t* num_rows_dev, int kv_heads,
                              int head_dim, void* k_codes, float* k_scales, int64_t k_rows, void* v_codes, float* v_scales,
                              int64_t v_rows, void* dv, void* stream) {
  int rc = check_heads("fp8_kv_cache_update", kv_heads, head_dim, batch, num_rows, k_rows < v_rows ? k_rows : v_rows);
  if (rc <= 0)
    return rc;
  if ((rc = check_stride("fp8_kv_cache_update", "k_new", k_new, ldk, kv_heads)) != DYLLM_OK ||
      (rc = check_stride("fp8_kv_cache_update", "v_new", v_new, ldv, kv_heads)) != DYLLM_OK)
    return rc;
  DYLLM_REQUIRE(max_pos > 0, DYLLM_ERR_INVALID_ARGUMENT, "fp8_kv_cache_update: an angle table of %d positions", max_pos);
  DYLLM_REQUIRE(rows_k && positions && cos_sin && cu_seqlens_k && k_seq_starts && v_seq_starts && seq_ids &&
                    ((k_codes && k_scales) || k_rows == 0) && ((v_codes && v_scales) || v_rows == 0) && dv,
                DYLLM_ERR_INVALID_ARGUMENT, "fp8_kv_cache_update: null pointer");
  DYLLM_REQUIRE(aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(dv, 16) && aligned(cos_sin, 16) &&
                    aligned(k_scales, 4) && aligned(v_scales, 4),
                DYLLM_ERR_INVALID_ARGUMENT, "fp8_kv_cache_update: codes, dv and cos_sin must be 16-byte aligned");
  auto launch = [&](auto groups) {
    constexpr int G = decltype(groups)::value;
    DYLLM_LAUNCH(fp8_kv_cache_update_kernel<G>, grid_of(num_rows, kv_heads, G), kThreads, 0, static_cast<cudaStream_t>(stream), static_cast<const uint4*>(k_new), ldk / 8, static_cast<const uint4*>(v_new), ldv / 8, rows_k, positions, pos_idx, reinterpret_cast<const float4*>(cos_sin), max_pos, cu_seqlens_k, k_seq_starts, v_seq_starts, seq_ids, batch, num_rows, num_rows_dev, kv_heads, static_cast<uint2*>(k_codes), k_scales, k_rows, static_cast<uint2*>(v_codes), v_scales, v_rows, static_cast<uint4*>(dv));
  };
  const int g = groups_of(num_rows, kv_heads, 2);
  g == 2 ? launch(Groups<2>()) : launch(Groups<1>());
  return check_launch("fp8_kv_cache_update");
}

}  // extern "C"
