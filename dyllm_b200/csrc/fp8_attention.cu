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

// s * log2(e) of one score, capped.
__device__ __forceinline__ float score_log2(float s, float cap) {
  if (cap > 0.f)      // tanh(x) = 1 - 2 / (1 + e^2x), absolute error a few 2^-24 (the hardware tanh has 2^-11)
    s = cap - 2.f * cap * __fdividef(1.f, 1.f + exp2f(__fdividef(2.f * kLog2e * s, cap)));
  return s * kLog2e;
}

// Exponent of a value's scale (a power of two by definition).
__device__ __forceinline__ float value_exponent(float scale) {
  const uint32_t bits = __float_as_uint(scale);
  if (bits >= 0x7f800000u)
    return __uint_as_float(0x7fc00000u);
  return static_cast<float>(max(static_cast<int>(bits >> 23) - 127, kFp8MinExp));
}

// ----------------------------------------------------------------------------------------------
// Few rows per sequence: bound by the bytes of the cache.  mma.sync on codes widened to half precision in registers.
//
// The rows of a tile are the (listed row, query head) pairs of one sequence and key head, 16 or 32 of them, so that grouped
// query heads share one pass over their keys.  A unit of work is 128 keys of a tile; all units of the launch, in the order
// (sequence, key head, tile, keys), are dealt out to the CTAs in equal contiguous shares that every CTA works out for itself
// from the device-side counts.  A tile whose units lie in several CTAs is joined by the CTA that finishes last, in the order
// of its parts.
//
// One producer warp feeds a ring of units (TMA boxes of 32 rows x 128 bytes, the scales by cp.async); each of four consumer
// warps takes 32 keys of a unit on its own (own running maximum and sum), and the four are joined when the tile ends.
//
// Operand layouts (g = lane / 4, c = lane % 4), chosen so that every shared-memory access is 16 bytes wide and the widening
// of four codes is one or two instructions per pair:
//   S = Q K^T    contraction step s = 0..7, thread c holds dimensions 32c + 4s .. +3 (two pairs) of key 8j + g: the 32 bytes
//                of a key that a thread needs are contiguous.
//   O = P V      output block nb = 0..15, column g is dimension 16g + nb: the 16 bytes of a key that a thread needs are
//                contiguous, and a byte permutation pairs two keys' codes.
// ----------------------------------------------------------------------------------------------
constexpr int kUnitKeys = 128;
constexpr uint32_t kKvBytes = kUnitKeys * kD;                                  // codes of K or V of a unit
constexpr uint32_t kScaleBytes = 2 * kUnitKeys * sizeof(float);
template <int RG>
struct FewCfg {
  static constexpr int kRing = 2 * RG;
  static constexpr int kThreads = 32 + 128 * RG;
  static constexpr uint32_t kMergeBytes = RG * 4 * 16 * kD * sizeof(float);
  static constexpr uint32_t kSmem = kRing * (2 * kKvBytes + kScaleBytes) + kMergeBytes + 1024;
};

struct FewParams {
  Fp8AttnParams a;
  const int2* spans;           // per sequence: keys that any of its listed rows sees (null: all)
  unsigned long long* tickets; // one per CTA
  float* parts;                // two per CTA: [rows][128] sums, [rows] maxima, [rows] sums of weights
  unsigned long long launch_id;
  int* status_word;
};

// Tickets of tiles whose parts lie in several CTAs, in a workspace that nobody has cleared: a word counts only once its upper
// 48 bits are this launch's number (any other content, also by chance one in 2^48, is replaced), and the last part leaves a
// zero, so that a launch that a graph replays finds it as if new.
__device__ __forceinline__ void open_join(unsigned long long* word, unsigned long long launch_id) {
  unsigned long long seen = *reinterpret_cast<volatile unsigned long long*>(word);
  while (((seen ^ launch_id) >> 16) != 0) {
    const unsigned long long was = atomicCAS(word, seen, launch_id);
    if (was == seen)
      return;
    seen = was;
  }
}
__device__ __forceinline__ bool last_to_join(unsigned long long* word, int parts) {
  if ((atomicAdd(word, 1ull) & 0xffff) != static_cast<unsigned long long>(parts - 1))
    return false;
  *reinterpret_cast<volatile unsigned long long*>(word) = 0;
  return true;
}

// A sequence as the work list sees it.
struct SeqWork {
  int b, row0, rows, tiles, units;      // rows: (listed row, head of the group) pairs
  int lo, hi;                           // keys
  int64_t k0, v0;
};
template <int MROWS>
__device__ __forceinline__ SeqWork seq_work(const FewParams& p, int b) {
  SeqWork w = {};
  w.b = b;
  if (b >= p.a.batch)
    return w;
  w.row0 = min(__ldg(p.a.cu_sal + b), p.a.num_salient);
  const int n = min(__ldg(p.a.cu_sal + b + 1), p.a.num_salient) - w.row0;
  if (n <= 0)
    return w;
  w.rows = n * (p.a.H / p.a.Hkv);
  const KeyRange kr = keys_of(p.a, b);
  w.k0 = kr.k0;
  w.v0 = kr.v0;
  w.hi = kr.len;
  if (p.spans) {
    const int2 s = __ldg(p.spans + b);
    w.lo = s.x;
    w.hi = s.y;
  }
  w.tiles = (w.rows + MROWS - 1) / MROWS;
  w.units = max(1, (w.hi - w.lo + kUnitKeys - 1) / kUnitKeys);
  return w;
}

// Walks over the parts of tiles that a CTA's share of the units consists of.  Uniform over a warp.
template <int MROWS>
struct Walk {
  SeqWork w;
  int64_t total, at, end, seq_first;    // units: of the launch, next, end of the share, first of the sequence
  int hk, tile, first, last;            // the part: units [first, last) of the tile
  int ctas;                             // CTAs that have a share
  int64_t tile_first;                   // first unit of the tile in the launch

  __device__ __forceinline__ void start(const FewParams& p) {
    const int lane = threadIdx.x & 31;
    int64_t sum = 0;
    for (int base = 0; base < p.a.batch; base += 32) {
      const SeqWork x = seq_work<MROWS>(p, base + lane);
      sum += static_cast<int64_t>(x.tiles) * x.units;
    }
#pragma unroll
    for (int s = 16; s; s >>= 1)
      sum += __shfl_xor_sync(0xffffffffu, sum, s);
    total = sum * p.a.Hkv;
    ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total));      // no share is empty
    at = end = 0;
    if (static_cast<int>(blockIdx.x) >= ctas)
      return;
    at = total * blockIdx.x / ctas;
    end = total * (blockIdx.x + 1) / ctas;
    seq_first = 0;
    for (int base = 0;; base += 32) {
      const SeqWork x = seq_work<MROWS>(p, base + lane);
      const int64_t mine = static_cast<int64_t>(x.tiles) * x.units * p.a.Hkv;
      int64_t scan = mine;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, scan, s);
        if (lane >= s)
          scan += o;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, seq_first + scan > at);
      if (hit) {
        const int src = __ffs(hit) - 1;
        seq_first += __shfl_sync(0xffffffffu, scan - mine, src);
        w = seq_work<MROWS>(p, base + src);
        return;
      }
      seq_first += __shfl_sync(0xffffffffu, scan, 31);
    }
  }
  // The next part, false at the end of the share.
  __device__ __forceinline__ bool next(const FewParams& p) {
    if (at >= end)
      return false;
    int64_t in_seq = at - seq_first;
    while (in_seq >= static_cast<int64_t>(w.tiles) * w.units * p.a.Hkv) {
      seq_first += static_cast<int64_t>(w.tiles) * w.units * p.a.Hkv;
      in_seq = at - seq_first;
      w = seq_work<MROWS>(p, w.b + 1);
    }
    const int t = static_cast<int>(in_seq / w.units);
    first = static_cast<int>(in_seq - static_cast<int64_t>(t) * w.units);
    hk = t / w.tiles;
    tile = t - hk * w.tiles;
    tile_first = at - first;
    last = static_cast<int>(min(static_cast<int64_t>(w.units), first + (end - at)));
    at += last - first;
    return true;
  }
  // CTA whose share holds unit u
  __device__ __forceinline__ int cta_of(int64_t u) const { return static_cast<int>(((u + 1) * ctas - 1) / total); }
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int RG>
__device__ __forceinline__ void consumers_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(128 * RG) : "memory");
}

// Power of two near 1 / amax and its inverse: queries go into half precision next to their row's largest element.
__device__ __forceinline__ float2 query_scales(uint32_t amax) {
  if (amax >= 0x7f800000u)
    return make_float2(__uint_as_float(0x7fc00000u), 1.f);
  const uint32_t e = min(max(amax >> 23, 1u), 252u);
  return make_float2(__uint_as_float((254u - e) << 23), __uint_as_float(e << 23));
}

// Sixteen values of output row t of a sequence's (listed row, head) pairs.
__device__ __forceinline__ void store_row(const FewParams& p, const SeqWork& w, int hk, int t, int oc, const float4 (&acc)[4], float sum,
                                          int group) {
  if (t >= w.rows)
    return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int i = t / group, h = hk * group + t - i * group;
  uint4* dst = reinterpret_cast<uint4*>(p.a.out + ((static_cast<int64_t>(w.row0) + i) * p.a.H + h) * kD) + oc / 2;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float x[8] = {acc[2 * j].x * inv, acc[2 * j].y * inv, acc[2 * j].z * inv, acc[2 * j].w * inv,
                        acc[2 * j + 1].x * inv, acc[2 * j + 1].y * inv, acc[2 * j + 1].z * inv, acc[2 * j + 1].w * inv};
    dst[j] = float_to_bf16x8(x);
  }
}

// RG: groups of 16 rows in a tile, four consumer warps each (RG = 2: one CTA per SM, twice the ring).
template <int RG, bool PLAIN>
__global__ void __launch_bounds__(FewCfg<RG>::kThreads, 3 - RG)
fp8_few_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const FewParams p) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  using Cfg = FewCfg<RG>;
  constexpr int MROWS = 16 * RG, kRing = Cfg::kRing;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_ring = smem;
  uint8_t* v_ring = smem + kRing * kKvBytes;
  float* merge = reinterpret_cast<float*>(smem + 2 * kRing * kKvBytes);
  float* scales = reinterpret_cast<float*>(smem + 2 * kRing * kKvBytes + Cfg::kMergeBytes);      // [stage][K, V][128]
  __shared__ uint64_t full[kRing], empty[kRing];
  __shared__ int abort_flag, joins;
  __shared__ float2 s_ml[4 * RG][16];      // (maximum, sum) of a warp's rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&full[i], 33);         // 32 lanes' scale copies and the bytes of the boxes
      mbar_init(&empty[i], 4 * RG);
    }
    fence_mbar_init();
  }
  __syncthreads();

  const Fp8AttnParams& a = p.a;
  Walk<MROWS> walk;
  walk.start(p);
  if (walk.at >= walk.end)
    return;

  if (warp == 4 * RG) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      tma_prefetch_desc(&tmap_k);
      tma_prefetch_desc(&tmap_v);
    }
    int n = 0;
    bool ok = true;
    while (ok && walk.next(p)) {
      const SeqWork& w = walk.w;
      if (w.hi <= w.lo)
        continue;
      for (int u = walk.first; ok && u < walk.last; ++u, ++n) {
        const int stage = n % kRing;
        if (n >= kRing && !mbar_wait(&empty[stage], (n / kRing - 1) & 1, &abort_flag, p.status_word, 401)) {
          ok = false;
          break;
        }
        const int key = w.lo + u * kUnitKeys;
        const int live = min(kUnitKeys, w.hi - key);
        uint8_t* ks = k_ring + stage * kKvBytes;
        uint8_t* vs = v_ring + stage * kKvBytes;
        if (lane == 0) {
          const int boxes = (live + 31) / 32;
          mbar_arrive_expect_tx(&full[stage], boxes * 2 * 32 * kD);
          for (int i = 0; i < boxes; ++i) {
            tma_load_2d(ks + i * 32 * kD, &tmap_k, &full[stage], walk.hk * kD, static_cast<int>(w.k0) + key + 32 * i);
            tma_load_2d(vs + i * 32 * kD, &tmap_v, &full[stage], walk.hk * kD, static_cast<int>(w.v0) + key + 32 * i);
          }
        }
        float* sc = scales + stage * 2 * kUnitKeys;
        const float* ksrc = a.k_scales + (w.k0 + key) * a.Hkv + walk.hk;
        const float* vsrc = a.v_scales + (w.v0 + key) * a.Hkv + walk.hk;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = lane + 32 * i;
          if (j < live) {
            cp_async4(sc + j, ksrc + static_cast<int64_t>(j) * a.Hkv);
            cp_async4(sc + kUnitKeys + j, vsrc + static_cast<int64_t>(j) * a.Hkv);
          }
        }
        cp_async_arrive(&full[stage]);
      }
    }
    // a CTA may not end with copies on their way, also when a wait of its consumers has given up
    for (int i = max(0, n - kRing); i < n; ++i)
      mbar_wait(&full[i % kRing], (i / kRing) & 1, &abort_flag, p.status_word, 402);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int g = lane >> 2, c = lane & 3;
  const int group = a.H / a.Hkv;
  const int rg = warp >> 2, slice = warp & 3;       // row group and 32 keys of a unit
  int n = 0;
  while (walk.next(p)) {
    const SeqWork w = walk.w;
    const int hk = walk.hk;
    // queries as A fragments
    uint32_t qf[8][4];
    float rf[2], slope[2];
    int pos[2], lo[2], hi[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int t = walk.tile * MROWS + rg * 16 + r * 8 + g;      // row of the sequence's (listed row, head) pairs
        const int i = t / group, h = hk * group + t - i * group;
        int row = -1;
        if (t < w.rows) {
          row = __ldg(a.idx + w.row0 + i);
          if (row >= a.total_q)
            row = -1;
        }
        uint4 x[4] = {};
        if (row >= 0) {
          const uint4* src = reinterpret_cast<const uint4*>(a.q + row * a.ldq + h * kD) + c * 4;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            x[j] = __ldg(src + j);
        }
        lo[r] = 0;
        hi[r] = row >= 0 ? w.hi : 0;
        pos[r] = 0;
        slope[r] = 0.f;
        if (!PLAIN && row >= 0) {
          pos[r] = __ldg(a.cu_k + w.b + 1) - __ldg(a.cu_k + w.b) - (__ldg(a.cu_q + w.b + 1) - row);
          if (a.slopes)
            slope[r] = __ldg(a.slopes + h) * kLog2e;
          if (a.ranges) {
            const int2 v = __ldg(a.ranges + row);
            lo[r] = v.x;
            hi[r] = min(v.y, w.hi);
          }
        }
        float y[32];
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          bf16x8_to_float(x[j], y + 8 * j);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const float2 qs = query_scales(m);
        rf[r] = qs.y * a.scale * (PLAIN ? kLog2e : 1.f);
#pragma unroll
        for (int st = 0; st < 8; ++st) {
          qf[st][r] = pack_half2(y[4 * st] * qs.x, y[4 * st + 1] * qs.x);
          qf[st][2 + r] = pack_half2(y[4 * st + 2] * qs.x, y[4 * st + 3] * qs.x);
        }
      }
    float o[16][4], mx[2], l[2];
#pragma unroll
      for (int nb = 0; nb < 16; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[nb][j] = 0.f;
      mx[0] = mx[1] = -INFINITY;
      l[0] = l[1] = 0.f;

    if (w.hi > w.lo) {
      for (int u = walk.first; u < walk.last; ++u, ++n) {
        const int stage = n % kRing;
        if (!mbar_wait(&full[stage], (n / kRing) & 1, &abort_flag, p.status_word, 403))
          break;
        const int key = w.lo + u * kUnitKeys + slice * 32;
        const int live = w.hi - key;                 // keys of this warp's 32 that exist
        if (live > 0) {
          const uint8_t* kt = k_ring + stage * kKvBytes + slice * 32 * kD;
          const uint8_t* vt = v_ring + stage * kKvBytes + slice * 32 * kD;
          const float* sc = scales + stage * 2 * kUnitKeys + slice * 32;
          float s[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 8 * j + g;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint4 x = *reinterpret_cast<const uint4*>(kt + r * kD + (((2 * c + half) ^ (r & 7)) << 4));
              const uint32_t wd[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t b0 = fp8_to_half2(wd[i] & 0xffffu), b1 = fp8_to_half2(wd[i] >> 16);
                  const uint32_t* q4 = qf[half * 4 + i];
                  mma_f16(s[j], q4[0], q4[1], q4[2], q4[3], b0, b1);
              }
            }
          }
          // scores, their maxima, weights
          uint32_t pf[4][2];
            float inv[4][2];
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 ks = *reinterpret_cast<const float2*>(sc + 8 * j + 2 * c);
              const float2 vs = *reinterpret_cast<const float2*>(sc + kUnitKeys + 8 * j + 2 * c);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float kscale = e ? ks.y : ks.x;
                const float ex = value_exponent(e ? vs.y : vs.x);
                inv[j][e] = __uint_as_float(static_cast<uint32_t>(127 - static_cast<int>(ex)) << 23);
                const int at = key + 8 * j + 2 * c + e;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  float t;
                  if (PLAIN) {
                    t = s[j][2 * r + e] * (kscale * rf[r]) + ex;
                    t = at < hi[r] ? t : -INFINITY;
                  } else {
                    t = score_log2(s[j][2 * r + e] * (kscale * rf[r]), a.cap) - slope[r] * static_cast<float>(abs(pos[r] - at)) + ex;
                    t = at >= lo[r] && at < hi[r] ? t : -INFINITY;
                  }
                  s[j][2 * r + e] = t;
                  top[r] = fmaxf(top[r], t);
                }
              }
            }
            float base[2], old[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
              top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
              top[r] = fmaxf(top[r], mx[r]);
              base[r] = top[r] == -INFINITY ? 0.f : top[r];
              old[r] = exp2f(mx[r] - base[r]);
            }
            if (__any_sync(0xffffffffu, top[0] > mx[0] || top[1] > mx[1])) {
#pragma unroll
              for (int nb = 0; nb < 16; ++nb) {
                o[nb][0] *= old[0];
                o[nb][1] *= old[0];
                o[nb][2] *= old[1];
                o[nb][3] *= old[1];
              }
              l[0] *= old[0];
              l[1] *= old[1];
              mx[0] = top[0];
              mx[1] = top[1];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                float p0 = exp2f(s[j][2 * r] - base[r]), p1 = exp2f(s[j][2 * r + 1] - base[r]);
                const int at = key + 8 * j + 2 * c;
                // the value scale of a key that does not exist is whatever the ring held: its weight is zero all the same
                l[r] += (at < w.hi ? p0 * inv[j][0] : 0.f) + (at + 1 < w.hi ? p1 * inv[j][1] : 0.f);
                pf[j][r] = pack_half2(p0, p1);
              }
          // O += P V
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = 16 * t + 2 * c + (i & 1) + (i >> 1) * 8;
              v[i] = *reinterpret_cast<const uint4*>(vt + r * kD + ((g ^ (r & 7)) << 4));
              if (live < 32 && r >= live)
                v[i] = make_uint4(0u, 0u, 0u, 0u);      // rows behind the last key may hold any byte
            }
            const uint32_t* v0 = &v[0].x;
            const uint32_t* v1 = &v[1].x;
            const uint32_t* v2 = &v[2].x;
            const uint32_t* v3 = &v[3].x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a01 = __byte_perm(v0[i], v1[i], 0x5140), a23 = __byte_perm(v0[i], v1[i], 0x7362);
              const uint32_t b01 = __byte_perm(v2[i], v3[i], 0x5140), b23 = __byte_perm(v2[i], v3[i], 0x7362);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t x0 = e < 2 ? a01 : a23, x1 = e < 2 ? b01 : b23;
                const uint32_t h0 = fp8_to_half2(e & 1 ? x0 >> 16 : x0 & 0xffffu);
                const uint32_t h1 = fp8_to_half2(e & 1 ? x1 >> 16 : x1 & 0xffffu);
                  mma_f16(o[4 * i + e], pf[2 * t][0], pf[2 * t][1], pf[2 * t + 1][0], pf[2 * t + 1][1], h0, h1);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&empty[stage]);
      }
    }

    // ---------------------------------------------------------------- join the four warps of a row group
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (c == 0)
        s_ml[warp][r * 8 + g] = make_float2(mx[r], l[r]);
    }
    consumers_sync<RG>();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = r * 8 + g;
      float top = s_ml[4 * rg][row].x;
#pragma unroll
      for (int i = 1; i < 4; ++i)
        top = fmaxf(top, s_ml[4 * rg + i][row].x);
      const float mul = exp2f(mx[r] - (top == -INFINITY ? 0.f : top));
      float* dst = merge + (warp * 16 + row) * kD;
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int chunk = 8 * c + 4 * e + i;
          *reinterpret_cast<float4*>(dst + ((chunk ^ (c + 4 * (g & 1))) << 2)) =
              make_float4(o[4 * i][2 * r + e] * mul, o[4 * i + 1][2 * r + e] * mul, o[4 * i + 2][2 * r + e] * mul,
                          o[4 * i + 3][2 * r + e] * mul);
        }
    }
    consumers_sync<RG>();
    // a thread's share of the result: a row of the tile, four chunks of four values
    const int orow = threadIdx.x >> 3, oc = (threadIdx.x & 7) * 4;
    const float2* ml = &s_ml[4 * (orow >> 4)][orow & 15];
    float top = ml[0].x;
#pragma unroll
    for (int i = 1; i < 4; ++i)
      top = fmaxf(top, ml[16 * i].x);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 acc[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum += ml[16 * i].y * exp2f(ml[16 * i].x - base);
      const float* src = merge + ((4 * (orow >> 4) + i) * 16 + (orow & 15)) * kD;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int chunk = oc + j;
        const float4 x = *reinterpret_cast<const float4*>(src + ((chunk ^ ((chunk >> 3) + 4 * (orow & 1))) << 2));
        acc[j].x += x.x;
        acc[j].y += x.y;
        acc[j].z += x.z;
        acc[j].w += x.w;
      }
    }
    const int owner = walk.cta_of(walk.tile_first);
    const int parts = walk.last - walk.first == w.units ? 1 : walk.cta_of(walk.tile_first + w.units - 1) - owner + 1;
    if (parts == 1) {
      store_row(p, w, hk, walk.tile * MROWS + orow, oc, acc, sum, group);
      consumers_sync<RG>();      // merge and s_ml are free again
      continue;
    }
    // ---------------------------------------------------------------- join the parts of a tile that several CTAs hold
    constexpr int kPart = MROWS * kD + 2 * MROWS;
    {
      float* part = p.parts + (2 * static_cast<int64_t>(blockIdx.x) + (walk.first == 0 ? 1 : 0)) * kPart;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(part + orow * kD + (oc + j) * 4) = acc[j];
      if (oc == 0) {
        part[MROWS * kD + orow] = top;
        part[MROWS * kD + MROWS + orow] = sum;
      }
    }
    __threadfence();
    consumers_sync<RG>();
    if (threadIdx.x == 0) {
      open_join(p.tickets + owner, p.launch_id);
      joins = last_to_join(p.tickets + owner, parts) ? 1 : 0;
    }
    consumers_sync<RG>();
    if (!joins)
      continue;
    __threadfence();
    top = -INFINITY;
    for (int i = 0; i < parts; ++i)
      top = fmaxf(top, __ldcg(p.parts + (2 * static_cast<int64_t>(owner + i) + (i == 0)) * kPart + MROWS * kD + orow));
    const float last_base = top == -INFINITY ? 0.f : top;
    sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int i = 0; i < parts; ++i) {
      const float* src = p.parts + (2 * static_cast<int64_t>(owner + i) + (i == 0)) * kPart;
      const float mul = exp2f(__ldcg(src + MROWS * kD + orow) - last_base);
      sum += __ldcg(src + MROWS * kD + MROWS + orow) * mul;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(src + orow * kD) + oc + j);
        acc[j].x += x.x * mul;
        acc[j].y += x.y * mul;
        acc[j].z += x.z * mul;
        acc[j].w += x.w * mul;
      }
    }
    store_row(p, w, hk, walk.tile * MROWS + orow, oc, acc, sum, group);
  }
}

// Keys that any listed row of a sequence sees; one warp per sequence.
__global__ void __launch_bounds__(128) fp8_spans_kernel(const Fp8AttnParams p, int2* __restrict__ spans) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  const int b = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (b >= p.batch)
    return;
  const int len = keys_of(p, b).len;
  int lo = len, hi = 0;
  for (int i = min(__ldg(p.cu_sal + b), p.num_salient) + (threadIdx.x & 31); i < min(__ldg(p.cu_sal + b + 1), p.num_salient); i += 32) {
    const int r = __ldg(p.idx + i);
    if (r < 0 || r >= p.total_q)
      continue;
    const int2 v = __ldg(p.ranges + r);
    const int x = max(v.x, 0), y = min(v.y, len);
    if (x < y) {
      lo = min(lo, x);
      hi = max(hi, y);
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if ((threadIdx.x & 31) == 0)
    spans[b] = lo < hi ? make_int2(lo, hi) : make_int2(0, 0);
}

size_t few_parts_offset(int batch, int ctas) {
  return (ctas * sizeof(unsigned long long) + batch * sizeof(int2) + 255) / 256 * 256;
}
size_t few_workspace(int batch, int ctas) {
  return few_parts_offset(batch, ctas) + 2ull * ctas * (32 * kD + 2 * 32) * sizeof(float);
}

template <int RG, bool PLAIN>
int launch_few(const CUtensorMap& tk, const CUtensorMap& tv, const FewParams& p, int ctas, cudaStream_t s) {
  static bool set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  dev = (dev < 0 || dev >= 64) ? 0 : dev;
  if (!set[dev]) {
    if (cudaFuncSetAttribute(fp8_few_rows_kernel<RG, PLAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(FewCfg<RG>::kSmem)) != cudaSuccess)
      return set_error(DYLLM_ERR_CUDA, "attention_salient_rows_fp8: cudaFuncSetAttribute failed: %s",
                       cudaGetErrorString(cudaGetLastError()));
    set[dev] = true;
  }
  DYLLM_LAUNCH((fp8_few_rows_kernel<RG, PLAIN>), RG == 1 ? ctas : ctas / 2, FewCfg<RG>::kThreads, FewCfg<RG>::kSmem, s, tk, tv, p);
  return check_launch("attention_salient_rows_fp8");
}

}  // namespace
}  // namespace dyllm

using namespace dyllm;

extern "C" {

size_t dyllm_attention_salient_rows_fp8_workspace_bytes(int num_salient, int batch, int num_heads, int num_kv_heads) {
  if (num_salient <= 0 || batch <= 0 || num_heads <= 0 || num_kv_heads <= 0)
    return 0;
  return few_workspace(batch, 2 * sm_count());
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
  DYLLM_REQUIRE(k_rows < (1ll << 31) && v_rows < (1ll << 31), DYLLM_ERR_UNSUPPORTED,
                "attention_salient_rows_fp8: caches of 2^31 rows or more");
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
  FewParams f = {};
  const int ctas = 2 * sm_count();
  DYLLM_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, DYLLM_ERR_INVALID_ARGUMENT,
                "attention_salient_rows_fp8: the workspace must be 16-byte aligned");
  DYLLM_REQUIRE(workspace && workspace_bytes >= few_workspace(batch, ctas), DYLLM_ERR_WORKSPACE,
                "attention_salient_rows_fp8: workspace of %zu bytes is smaller than the %zu required", workspace_bytes,
                few_workspace(batch, ctas));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  f.a = p;
  f.tickets = reinterpret_cast<unsigned long long*>(ws);
  int2* spans = reinterpret_cast<int2*>(ws + ctas * sizeof(unsigned long long));
  f.parts = reinterpret_cast<float*>(ws + few_parts_offset(batch, ctas));
  f.launch_id = next_launch_id() & ~0xffffull;
  f.status_word = device_status_word();
  if (p.ranges) {
    f.spans = spans;
    DYLLM_LAUNCH(fp8_spans_kernel, cdiv_i(batch, 4), 128, 0, st, p, spans);
  }
  CUtensorMap tk, tv;
  const uint64_t width = static_cast<uint64_t>(num_kv_heads) * kD;
  int rc = encode_tmap_2d_u8(&tk, k_codes, k_rows ? k_rows : 1, width, width, 32, kD);
  if (rc == DYLLM_OK)
    rc = encode_tmap_2d_u8(&tv, v_codes, v_rows ? v_rows : 1, width, width, 32, kD);
  if (rc != DYLLM_OK)
    return rc;
  const bool plain = softcap == 0.f && !slopes && !key_ranges;
  const bool one = static_cast<int64_t>(max_rows_per_seq) * (num_heads / num_kv_heads) <= 16;
  if (one)
    rc = plain ? launch_few<1, true>(tk, tv, f, ctas, st) : launch_few<1, false>(tk, tv, f, ctas, st);
  else
    rc = plain ? launch_few<2, true>(tk, tv, f, ctas, st) : launch_few<2, false>(tk, tv, f, ctas, st);
  return rc;
}

}  // extern "C"
