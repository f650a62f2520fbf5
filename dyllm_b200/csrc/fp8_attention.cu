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
// Few rows per sequence: bound by the bytes of the cache, which go from the TMA ring to the tensor cores as they are.
//
// The rows of a tile are the (listed row, query head) pairs of one sequence and key head, RN = 16 or 32 of them, so that
// grouped query heads share one pass over their keys.  A unit of work is 128 keys of a tile; all units of the launch, in the
// order (sequence, key head, tile, keys), are dealt out to the CTAs in equal contiguous shares that every CTA works out for
// itself from the device-side counts.  A tile whose units lie in several CTAs is joined by the CTA that finishes last, in the
// order of its parts.
//
// The products are transposed, keys (then head dimensions) in the M = 128 of tcgen05.mma.kind::f8f6f4:
//   S^T = K Q^T         A: K tile as loaded (K-major), B: the queries as e4m3 + e5m2, two products into one accumulator
//   O^T = V^T P^T       A: V tile as loaded (MN-major), B: the weights, 32 columns of e4m3 and 32 of their remainders
// A query in bf16 (8 significant bits) is e4m3 (4 bits) plus a remainder of at most 3 bits, which e5m2 holds exactly down to
// 2^-25 of the row's largest element.  A weight in [0, 1] is taken as e4m3(256 w) + e4m3(16 * remainder) / 16: off by at most
// 2^-8 of itself, or 2^-22.  The codes of the cache are never widened.
//
// Softmax per chunk of up to kChunk tiles: thread = key, first the scores of all tiles of the chunk (kept in tensor memory in
// place of the products) and their maxima, then weights tile by tile; the sums are rescaled between chunks.  Eight softmax
// warps, two per quarter of the keys, each with half of the rows; a TMA warp and an MMA warp.  Two CTAs per SM.
// ----------------------------------------------------------------------------------------------
constexpr int kUnitKeys = 128;
constexpr int kRing = 4;                                     // slots of one K or V tile
constexpr uint32_t kTileBytes = kUnitKeys * kD;
constexpr int kFewThreads = 320;
constexpr uint32_t kTmemCols = 256;
template <int RN>
struct FewCfg {
  static constexpr int kHalf = RN / 2;                       // rows of a softmax warp
  static constexpr int kChunk = RN == 16 ? 8 : 6;
  static constexpr uint32_t kTmemO = kChunk * RN;            // columns of O^T behind those of S^T: RN of 256 w, RN of remainders
  static constexpr uint32_t kQBytes = RN * kD;
  static constexpr uint32_t kSmem = (kRing + 2) * kTileBytes + 2 * kQBytes + 1024;
  static_assert(kTmemO + 2 * RN <= kTmemCols, "tensor memory of two CTAs per SM");
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
  int64_t total, left;                  // units: of the launch, of the share that are still to come
  int64_t tile_first;                   // first unit of the tile in the launch
  int hk, tile, first, last;            // the part: units [first, last) of the tile
  int ctas;                             // CTAs that have a share
  bool begun;

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
    left = 0;
    begun = false;
    if (static_cast<int>(blockIdx.x) >= ctas)
      return;
    const int64_t at = share(blockIdx.x);
    left = share(blockIdx.x + 1) - at;
    int64_t before = 0;
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
      const unsigned hit = __ballot_sync(0xffffffffu, before + scan > at);
      if (hit) {
        const int src = __ffs(hit) - 1;
        before += __shfl_sync(0xffffffffu, scan - mine, src);
        w = seq_work<MROWS>(p, base + src);
        break;
      }
      before += __shfl_sync(0xffffffffu, scan, 31);
    }
    const int64_t t = (at - before) / w.units;
    first = static_cast<int>(at - before - t * w.units);
    tile_first = at - first;
    hk = static_cast<int>(t / w.tiles);
    tile = static_cast<int>(t - static_cast<int64_t>(hk) * w.tiles);
  }
  // The next part, false at the end of the share.
  __device__ __forceinline__ bool next(const FewParams& p) {
    if (left == 0)
      return false;
    if (begun) {
      first = 0;
      tile_first += w.units;
      if (++tile == w.tiles) {
        tile = 0;
        if (++hk == p.a.Hkv) {
          hk = 0;
          do
            w = seq_work<MROWS>(p, w.b + 1);
          while (w.tiles == 0);
        }
      }
    }
    begun = true;
    last = static_cast<int>(min(static_cast<int64_t>(w.units), first + left));
    left -= last - first;
    return true;
  }
  // First unit of a CTA's share, and the CTA whose share holds unit u.
  __device__ __forceinline__ int64_t share(int64_t cta) const { return total * cta / ctas; }
  __device__ __forceinline__ int cta_of(int64_t u) const { return static_cast<int>(((u + 1) * ctas - 1) / total); }
};

// One arrival for the warp, after what all of its lanes have done (an arrival per lane is a shared-memory atomic each).
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0)
    mbar_arrive(bar);
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Maximum or sum of each of N = 8 or 16 values over the lanes of a warp: lane l gets that of value l / (32 / N).
template <int N, bool MAX>
__device__ __forceinline__ float reduce_lanes(const float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  auto join = [](float x, float y) { return MAX ? fmaxf(x, y) : x + y; };
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    x[i] = v[i];
  int bit = 16;
#pragma unroll
  for (int n = N / 2; n >= 1; n >>= 1, bit >>= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      if (i < n) {
        const float keep = up ? x[i + n] : x[i], give = up ? x[i] : x[i + n];
        x[i] = join(keep, __shfl_xor_sync(0xffffffffu, give, bit));
      }
  }
#pragma unroll
  for (int b = 16 / N; b >= 1; b >>= 1)
    x[0] = join(x[0], __shfl_xor_sync(0xffffffffu, x[0], b));
  return x[0];
}

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[N]) {
  if constexpr (N == 16)
    tmem_ld_32x16(addr, r);
  else
    tmem_ld_32x8(addr, r);
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[N]) {
  if constexpr (N == 16)
    tmem_st_32x16(addr, r);
  else
    tmem_st_32x8(addr, r);
}
// N consecutive floats of shared memory, 16-byte aligned, the same for all lanes
template <int N>
__device__ __forceinline__ void lds_row(float (&x)[N], const float* src) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(src + 4 * i);
    x[4 * i] = v.x;
    x[4 * i + 1] = v.y;
    x[4 * i + 2] = v.z;
    x[4 * i + 3] = v.w;
  }
}

// Keys of a part: [begin, end), in tiles from begin on.
template <int RN>
__device__ __forceinline__ int2 part_keys(const Walk<RN>& walk) {
  const int begin = walk.w.lo + walk.first * kUnitKeys;
  return make_int2(begin, min(walk.w.hi, walk.w.lo + walk.last * kUnitKeys));
}

template <int RN, bool PLAIN>
__global__ void __launch_bounds__(kFewThreads, 2)
fp8_few_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const FewParams p) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  using Cfg = FewCfg<RN>;
  constexpr int HR = Cfg::kHalf, kChunk = Cfg::kChunk;
  const Fp8AttnParams& a = p.a;
  Walk<RN> walk;
  walk.start(p);
  if (walk.left == 0)
    return;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* p_smem = ring + kRing * kTileBytes;               // two slots of [128 keys][128 bytes]: weights, then remainders
  uint8_t* q_smem = p_smem + 2 * kTileBytes;                 // [RN][128] e4m3, then e5m2
  __shared__ uint64_t full[kRing], empty[kRing], s_full[kChunk], p_full[2], p_free[2], q_full, s_free, pv_done, o_free;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, joins;
  __shared__ __align__(16) float s_rf[RN], s_slope[RN], s_max[4][RN], s_sum[4][RN];
  __shared__ int s_pos[RN];
  __shared__ int64_t s_out[RN];
  __shared__ int2 s_range[RN];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kChunk; ++i)
      mbar_init(&s_full[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&p_full[i], 8);
      mbar_init(&p_free[i], 1);
    }
    mbar_init(&q_full, 8);
    mbar_init(&s_free, 8);
    mbar_init(&pv_done, 1);
    mbar_init(&o_free, 8);
    fence_mbar_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_s = tmem_slot, tmem_o = tmem_slot + Cfg::kTmemO;

  if (warp == 0) {
    // ---------------------------------------------------------------- producer: K tiles of a chunk, then its V tiles
    int n = 0;
    while (walk.next(p)) {
      const SeqWork& w = walk.w;
      if (w.hi <= w.lo)
        continue;
      const int2 keys = part_keys(walk);
      const int tiles = (keys.y - keys.x + kUnitKeys - 1) / kUnitKeys;
      for (int c0 = 0; c0 < tiles; c0 += kChunk) {
        const int nt = min(kChunk, tiles - c0);
        for (int i = 0; i < 2 * nt; ++i, ++n) {
          const int slot = n % kRing;
          if (n >= kRing)
            mbar_wait(&empty[slot], (n / kRing - 1) & 1, &abort_flag, p.status_word, 401);
          if (lane == 0) {
            const CUtensorMap* map = i < nt ? &tmap_k : &tmap_v;
            const int key = keys.x + (c0 + (i < nt ? i : i - nt)) * kUnitKeys;
            const int row = static_cast<int>(i < nt ? w.k0 : w.v0) + key;
            const int boxes = min(4, (keys.y - key + 31) / 32);      // no box of keys that do not belong to the part
            mbar_arrive_expect_tx(&full[slot], boxes * 32 * kD);
            for (int j = 0; j < boxes; ++j)
              tma_load_2d(ring + slot * kTileBytes + j * 32 * kD, map, &full[slot], walk.hk * kD, row + 32 * j);
          }
          __syncwarp();
        }
      }
    }
    // a CTA may not end with copies on their way, also when a wait of another warp has given up
    for (int i = max(0, n - kRing); i < n; ++i)
      mbar_wait(&full[i % kRing], (i / kRing) & 1, &abort_flag, p.status_word, 402);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc_hi = umma_idesc_f8(128, RN, 0, 0, 0, 0), idesc_lo = umma_idesc_f8(128, RN, 0, 1, 0, 0);
    constexpr uint32_t idesc_pv = umma_idesc_f8(128, 2 * RN, 0, 0, 1, 1);
    const uint32_t q_addr = smem_u32(q_smem);
    int n = 0, n_p = 0, n_chunk = 0, n_part = 0;
    while (walk.next(p)) {
      const SeqWork& w = walk.w;
      if (w.hi <= w.lo)
        continue;
      const int2 keys = part_keys(walk);
      const int tiles = (keys.y - keys.x + kUnitKeys - 1) / kUnitKeys;
      mbar_wait(&q_full, n_part & 1, &abort_flag, p.status_word, 403);
      for (int c0 = 0; c0 < tiles; c0 += kChunk, ++n_chunk) {
        const int nt = min(kChunk, tiles - c0);
        if (n_chunk > 0)
          mbar_wait(&s_free, (n_chunk - 1) & 1, &abort_flag, p.status_word, 404);
        for (int i = 0; i < nt; ++i, ++n) {
          const int slot = n % kRing;
          mbar_wait(&full[slot], (n / kRing) & 1, &abort_flag, p.status_word, 405);
          tc_fence_after_sync();
          if (lane == 0) {
            const uint64_t a_desc = umma_smem_desc_sw128(smem_u32(ring + slot * kTileBytes), 16, 1024);
            const uint64_t hi_desc = umma_smem_desc_sw128(q_addr, 16, 1024);
            const uint64_t lo_desc = umma_smem_desc_sw128(q_addr + Cfg::kQBytes, 16, 1024);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {      // 32 head dimensions = 32 bytes a step
              umma_ss_f8(tmem_s + i * RN, a_desc + 2 * kk, hi_desc + 2 * kk, idesc_hi, kk != 0 ? 1u : 0u);
              umma_ss_f8(tmem_s + i * RN, a_desc + 2 * kk, lo_desc + 2 * kk, idesc_lo, 1u);
            }
            umma_commit(&empty[slot]);
            umma_commit(&s_full[i]);
          }
          __syncwarp();
        }
        for (int i = 0; i < nt; ++i, ++n, ++n_p) {
          const int slot = n % kRing, buf = n_p & 1;
          mbar_wait(&full[slot], (n / kRing) & 1, &abort_flag, p.status_word, 406);
          mbar_wait(&p_full[buf], (n_p >> 1) & 1, &abort_flag, p.status_word, 407);
          if (c0 == 0 && i == 0 && n_part > 0)
            mbar_wait(&o_free, (n_part - 1) & 1, &abort_flag, p.status_word, 408);
          tc_fence_after_sync();
          if (lane == 0) {
            const uint32_t v_addr = smem_u32(ring + slot * kTileBytes), p_addr = smem_u32(p_smem + buf * kTileBytes);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)        // 32 keys = 32 rows of 128 bytes a step
              umma_ss_f8(tmem_o, umma_smem_desc_sw128(v_addr + kk * 4096, kTileBytes, 1024),
                         umma_smem_desc_sw128(p_addr + kk * 4096, kTileBytes, 1024), idesc_pv, (c0 | i | kk) != 0 ? 1u : 0u);
            umma_commit(&empty[slot]);
            umma_commit(&p_free[buf]);
            if (i == nt - 1)
              umma_commit(&pv_done);
          }
          __syncwarp();
        }
      }
      ++n_part;
    }
  } else {
    // ---------------------------------------------------------------- softmax over the keys, epilogue
    const int half = (warp - 2) >> 2;              // rows HR * half ..
    const int quarter = warp & 3;                  // tensor-memory lanes: keys (head dimensions) 32 * quarter ..
    const int tid = threadIdx.x - 64;
    const int kl = quarter * 32 + lane;            // key of a tile, or head dimension
    const uint32_t t_lane = static_cast<uint32_t>(quarter * 32) << 16;
    const int group = a.H / a.Hkv;
    const int r0 = half * HR;
    uint32_t s_phase = 0;                          // bit i: phase of s_full[i]
    int n = 0, n_p = 0, n_chunk = 0;
    while (walk.next(p)) {
      const SeqWork w = walk.w;
      const int hk = walk.hk;
      if (w.hi <= w.lo) {                          // no keys: zeros
        for (int r = r0; r < r0 + HR && walk.tile * RN + r < w.rows; ++r) {
          const int t = walk.tile * RN + r, i = t / group;
          a.out[((static_cast<int64_t>(w.row0) + i) * a.H + hk * group + t - i * group) * kD + kl] = __float2bfloat16_rn(0.f);
        }
        continue;
      }
      // queries to shared memory; eight threads a row
      if (tid < RN * 8) {
        const int r = tid >> 3, part = tid & 7;
        const int t = walk.tile * RN + r, i = t / group, h = hk * group + t - i * group;
        int row = t < w.rows ? __ldg(a.idx + w.row0 + i) : -1;
        if (row >= a.total_q)
          row = -1;
        uint4 x0 = make_uint4(0u, 0u, 0u, 0u), x1 = x0;
        if (row >= 0) {
          const uint4* src = reinterpret_cast<const uint4*>(a.q + row * a.ldq + h * kD) + part * 2;
          x0 = __ldg(src);
          x1 = __ldg(src + 1);
        }
        float y[16];
        bf16x8_to_float(x0, y);
        bf16x8_to_float(x1, y + 8);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
        const uint32_t scale = fp8_scale_bits(fp8_amax8(m));
        const float inv = fp8_inverse(scale);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float z[4], e[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            z[k] = scale >= 0x7f800000u ? 0.f : y[4 * j + k] * inv;
          hi[j] = fp8_pack2(z[0], z[1]) | fp8_pack2(z[2], z[3]) << 16;
          const float2 u = fp8_to_float2(hi[j] & 0xffffu), v = fp8_to_float2(hi[j] >> 16);
          e[0] = z[0] - u.x, e[1] = z[1] - u.y, e[2] = z[2] - v.x, e[3] = z[3] - v.y;
          lo[j] = fp8_pack2_e5m2(e[0], e[1]) | fp8_pack2_e5m2(e[2], e[3]) << 16;
        }
        uint8_t* dst = q_smem + r * kD + ((part ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(dst + Cfg::kQBytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if (part == 0) {
          s_rf[r] = __uint_as_float(scale);        // NaN: a query that is not finite
          // output row, negative: none; the lowest bit: whether the row exists in q
          s_out[r] = t < w.rows ? ((static_cast<int64_t>(w.row0) + i) * a.H + h) * 2 + (row >= 0) : -1;
          if (!PLAIN) {
            s_pos[r] = __ldg(a.cu_k + w.b + 1) - __ldg(a.cu_k + w.b) - (__ldg(a.cu_q + w.b + 1) - row);
            s_slope[r] = a.slopes && row >= 0 ? __ldg(a.slopes + h) * kLog2e : 0.f;
            int2 v = make_int2(0, row >= 0 ? w.hi : 0);
            if (a.ranges && row >= 0) {
              v = __ldg(a.ranges + row);
              v.y = min(v.y, w.hi);
            }
            s_range[r] = v;
          }
        }
        fence_proxy_async_smem();
      }
      warp_arrive(&q_full);
      softmax_sync();

      const int2 keys = part_keys(walk);
      const int tiles = (keys.y - keys.x + kUnitKeys - 1) / kUnitKeys;
      const float* k_scale = a.k_scales + w.k0 * a.Hkv + hk;
      const float* v_scale = a.v_scales + w.v0 * a.Hkv + hk;
      float top[HR], l[HR];
#pragma unroll
      for (int r = 0; r < HR; ++r) {
        top[r] = -INFINITY;
        l[r] = 0.f;
      }
      for (int c0 = 0; c0 < tiles; c0 += kChunk, ++n_chunk) {
        const int nt = min(kChunk, tiles - c0);
        const int key0 = keys.x + c0 * kUnitKeys + kl;
        // scores of all tiles of the chunk, their maxima
        float mx[HR];
#pragma unroll
        for (int r = 0; r < HR; ++r)
          mx[r] = -INFINITY;
        {
          float rf[HR];
          lds_row(rf, s_rf + r0);
          float ks_next = 0.f, vs_next = 1.f;
          if (key0 < keys.y) {
            ks_next = __ldg(k_scale + static_cast<int64_t>(key0) * a.Hkv);
            vs_next = __ldg(v_scale + static_cast<int64_t>(key0) * a.Hkv);
          }
          for (int i = 0; i < nt; ++i) {
            const int at = key0 + i * kUnitKeys;
            const bool there = at < keys.y;
            const float kk = ks_next * a.scale * (PLAIN ? kLog2e : 1.f), ex = value_exponent(vs_next);
            if (at + kUnitKeys < keys.y) {
              ks_next = __ldg(k_scale + static_cast<int64_t>(at + kUnitKeys) * a.Hkv);
              vs_next = __ldg(v_scale + static_cast<int64_t>(at + kUnitKeys) * a.Hkv);
            }
            mbar_wait(&s_full[i], (s_phase >> i) & 1, &abort_flag, p.status_word, 409);
            tc_fence_after_sync();
            uint32_t s[HR];
            tmem_ld(tmem_s + t_lane + i * RN + r0, s);
            tmem_ld_wait();
#pragma unroll
            for (int r = 0; r < HR; ++r) {
              float t = __uint_as_float(s[r]) * (kk * rf[r]);
              if (PLAIN) {
                t += ex;
                t = there ? t : -INFINITY;
              } else {
                const int2 range = s_range[r0 + r];
                t = score_log2(t, a.cap) - s_slope[r0 + r] * static_cast<float>(abs(s_pos[r0 + r] - at)) + ex;
                t = there && at >= range.x && at < range.y ? t : -INFINITY;
              }
              s[r] = __float_as_uint(t);
              mx[r] = fmaxf(mx[r], t);
            }
            tmem_st(tmem_s + t_lane + i * RN + r0, s);
          }
          s_phase ^= (1u << nt) - 1;
        }
        tmem_st_wait();
        {
          const float v = reduce_lanes<HR, true>(mx);
          if (lane % (32 / HR) == 0)
            s_max[quarter][r0 + lane / (32 / HR)] = v;
        }
        softmax_sync();
        bool grown = false;
        float old[HR];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          float x[HR];
          lds_row(x, s_max[q4] + r0);
#pragma unroll
          for (int r = 0; r < HR; ++r)
            mx[r] = q4 == 0 ? fmaxf(x[r], top[r]) : fmaxf(mx[r], x[r]);
        }
#pragma unroll
        for (int r = 0; r < HR; ++r) {
          grown = grown || mx[r] > top[r];
          old[r] = exp2f(top[r] - (mx[r] == -INFINITY ? 0.f : mx[r]));
          top[r] = mx[r];
          l[r] *= old[r];
        }
        if (c0 > 0)      // every phase is waited for, also where nothing is rescaled
          mbar_wait(&pv_done, (n_chunk - 1) & 1, &abort_flag, p.status_word, 410);
        if (c0 > 0 && grown) {      // the same rows in all four quarters
          tc_fence_after_sync();
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t o[HR];
            tmem_ld(tmem_o + t_lane + j * RN + r0, o);
            tmem_ld_wait();
#pragma unroll
            for (int r = 0; r < HR; ++r)
              o[r] = __float_as_uint(__uint_as_float(o[r]) * old[r]);
            tmem_st(tmem_o + t_lane + j * RN + r0, o);
          }
          tmem_st_wait();
        }
        // weights
        for (int i = 0; i < nt; ++i, ++n_p) {
          const int at = key0 + i * kUnitKeys, buf = n_p & 1;
          uint32_t s[HR];
          tmem_ld(tmem_s + t_lane + i * RN + r0, s);
          float inv = 0.f;
          if (at < keys.y) {
            const float ex = value_exponent(__ldg(v_scale + static_cast<int64_t>(at) * a.Hkv));
            inv = ex == ex ? exp2f(-ex) : 1.f;      // the weight of a NaN is a NaN where the key is seen, else zero
          }
          tmem_ld_wait();
          if (n_p >= 2)
            mbar_wait(&p_free[buf], ((n_p >> 1) - 1) & 1, &abort_flag, p.status_word, 411);
          uint32_t hi[HR / 4], lo[HR / 4];
#pragma unroll
          for (int j = 0; j < HR / 4; ++j) {
            float w4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = 4 * j + k;
              w4[k] = exp2f(__uint_as_float(s[r]) + (8.f - (top[r] == -INFINITY ? 0.f : top[r])));
              l[r] += at < keys.y ? w4[k] * inv : 0.f;
            }
            hi[j] = fp8_pack2(w4[0], w4[1]) | fp8_pack2(w4[2], w4[3]) << 16;
            const float2 u = fp8_to_float2(hi[j] & 0xffffu), v = fp8_to_float2(hi[j] >> 16);
            lo[j] = fp8_pack2(16.f * w4[0] - 16.f * u.x, 16.f * w4[1] - 16.f * u.y) |
                    fp8_pack2(16.f * w4[2] - 16.f * v.x, 16.f * w4[3] - 16.f * v.y) << 16;
          }
          // row kl of the slot: RN weights, then RN remainders, in 16-byte chunks that the swizzle permutes
          uint8_t* dst = p_smem + buf * kTileBytes + kl * kD;
          if constexpr (HR == 16) {
            *reinterpret_cast<uint4*>(dst + ((half ^ (kl & 7)) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(dst + (((2 + half) ^ (kl & 7)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          } else {
            *reinterpret_cast<uint2*>(dst + ((0 ^ (kl & 7)) << 4) + 8 * half) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(dst + ((1 ^ (kl & 7)) << 4) + 8 * half) = make_uint2(lo[0], lo[1]);
          }
          if (keys.y - (key0 - kl) - i * kUnitKeys < kUnitKeys && half == 0) {
            // rows behind the last key may hold any byte, a NaN times a weight of zero among them
            const int use = n + nt + i;
            mbar_wait(&full[use % kRing], (use / kRing) & 1, &abort_flag, p.status_word, 412);
            if (at >= keys.y) {
              uint4* v = reinterpret_cast<uint4*>(ring + (use % kRing) * kTileBytes + kl * kD);
#pragma unroll
              for (int j = 0; j < 8; ++j)
                v[j] = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          tc_fence_before_sync();
          fence_proxy_async_smem();
          warp_arrive(&p_full[buf]);
        }
        warp_arrive(&s_free);
        n += 2 * nt;
      }

      // ---------------------------------------------------------------- thread = head dimension kl of HR rows
      {
        const float v = reduce_lanes<HR, false>(l);
        if (lane % (32 / HR) == 0)
          s_sum[quarter][r0 + lane / (32 / HR)] = v;
      }
      softmax_sync();
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        float x[HR];
        lds_row(x, s_sum[q4] + r0);
#pragma unroll
        for (int r = 0; r < HR; ++r)
          l[r] = q4 == 0 ? x[r] : l[r] + x[r];
      }
      mbar_wait(&pv_done, (n_chunk - 1) & 1, &abort_flag, p.status_word, 413);
      tc_fence_after_sync();
      float o[HR];
      {
        uint32_t u[HR], v[HR];
        tmem_ld(tmem_o + t_lane + r0, u);
        tmem_ld(tmem_o + t_lane + RN + r0, v);
        tmem_ld_wait();
#pragma unroll
        for (int r = 0; r < HR; ++r)
          o[r] = __uint_as_float(u[r]) + __uint_as_float(v[r]) * 0.0625f;
      }
      tc_fence_before_sync();
      warp_arrive(&o_free);

      bool store = walk.last - walk.first == w.units;
      if (!store) {
        const int owner = walk.first == 0 ? blockIdx.x : walk.cta_of(walk.tile_first);
        const int parts = walk.cta_of(walk.tile_first + w.units - 1) - owner + 1;
        // join the parts of a tile that several CTAs hold
        constexpr int kPart = RN * kD + 2 * RN;
        float* part = p.parts + (2 * static_cast<int64_t>(blockIdx.x) + (walk.first == 0 ? 1 : 0)) * kPart;
#pragma unroll
        for (int r = 0; r < HR; ++r)
          part[(r0 + r) * kD + kl] = o[r];
        if (kl == 0) {
#pragma unroll
          for (int r = 0; r < HR; ++r) {
            part[RN * kD + r0 + r] = top[r];
            part[RN * kD + RN + r0 + r] = l[r];
          }
        }
        __threadfence();
        softmax_sync();
        if (tid == 0) {
          open_join(p.tickets + owner, p.launch_id);
          joins = last_to_join(p.tickets + owner, parts) ? 1 : 0;
        }
        softmax_sync();
        store = joins;
        if (store) {
          __threadfence();
          const float* first = p.parts + (2 * static_cast<int64_t>(owner) + 1) * kPart;
          const float* rest = p.parts + 2 * static_cast<int64_t>(owner) * kPart;
#pragma unroll
          for (int r = 0; r < HR; ++r) {
            top[r] = -INFINITY;
            o[r] = l[r] = 0.f;
          }
          for (int i = 0; i < parts; ++i) {
            const float* src = i == 0 ? first : rest + 2 * static_cast<int64_t>(i) * kPart;
#pragma unroll
            for (int r = 0; r < HR; ++r)
              top[r] = fmaxf(top[r], __ldcg(src + RN * kD + r0 + r));
          }
          for (int i = 0; i < parts; ++i) {
            const float* src = i == 0 ? first : rest + 2 * static_cast<int64_t>(i) * kPart;
#pragma unroll
            for (int r = 0; r < HR; ++r) {
              const float mul = exp2f(__ldcg(src + RN * kD + r0 + r) - (top[r] == -INFINITY ? 0.f : top[r]));
              l[r] += __ldcg(src + RN * kD + RN + r0 + r) * mul;
              o[r] += __ldcg(src + (r0 + r) * kD + kl) * mul;
            }
          }
        }
      }
      if (store) {
#pragma unroll
        for (int r = 0; r < HR; ++r) {
          const int64_t at = s_out[r0 + r];
          if (at >= 0)
            a.out[(at >> 1) * kD + kl] = __float2bfloat16_rn(l[r] == 0.f || !(at & 1) ? 0.f : o[r] * __fdividef(1.f, l[r]));
        }
      }
      softmax_sync();      // what describes the rows is free again
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_slot, kTmemCols);
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

template <int RN, bool PLAIN>
int launch_few(const CUtensorMap& tk, const CUtensorMap& tv, const FewParams& p, int ctas, cudaStream_t s) {
  static bool set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  dev = (dev < 0 || dev >= 64) ? 0 : dev;
  if (!set[dev]) {
    if (cudaFuncSetAttribute(fp8_few_rows_kernel<RN, PLAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(FewCfg<RN>::kSmem)) != cudaSuccess)
      return set_error(DYLLM_ERR_CUDA, "attention_salient_rows_fp8: cudaFuncSetAttribute failed: %s",
                       cudaGetErrorString(cudaGetLastError()));
    set[dev] = true;
  }
  DYLLM_LAUNCH((fp8_few_rows_kernel<RN, PLAIN>), ctas, kFewThreads, FewCfg<RN>::kSmem, s, tk, tv, p);
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
    rc = plain ? launch_few<16, true>(tk, tv, f, ctas, st) : launch_few<16, false>(tk, tv, f, ctas, st);
  else
    rc = plain ? launch_few<32, true>(tk, tv, f, ctas, st) : launch_few<32, false>(tk, tv, f, ctas, st);
  return rc;
}

}  // extern "C"
