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

// cap * tanh(s / cap) from z = 2 log2(e) s / cap: tanh(x) = 1 - 2 / (1 + e^2x), absolute error a few 2^-24 (the hardware tanh
// has 2^-11).
__device__ __forceinline__ float capped(float z, float cap) { return cap - 2.f * cap * __fdividef(1.f, 1.f + exp2f(z)); }

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
constexpr int kRows = 32, kGroup = 8;                        // rows of a tile, of a softmax warp
constexpr int kChunk = 4;                                    // tiles whose scores are in registers at a time
constexpr int kRing = 8;                                     // slots of one K or V tile
constexpr int kParts = 4;                                    // slots of part descriptions
constexpr uint32_t kTileBytes = kUnitKeys * kD, kQBytes = kRows * kD;
constexpr int kSoftmaxWarps = 16, kFewThreads = 32 * (kSoftmaxWarps + 3);
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kFewSmem = (kRing + kChunk / 2) * kTileBytes + 4 * kQBytes + 2 * kChunk * 2 * kUnitKeys * sizeof(float) + 1024;

struct FewParams {
  Fp8AttnParams a;
  const int2* spans;           // per tile of rows: keys that any of them sees (null: all)
  unsigned long long* tickets; // one per CTA
  float* parts;                // two per CTA: [rows][128] sums, [rows] maxima, [rows] sums of weights
  int* joins;                  // many rows, per CTA: parts of the tile that begins in it and goes on in others (0: none)
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
  int b, row0, rows, tiles;             // rows: (listed row, head of the group) pairs
  int len;                              // keys
  int k0, v0;                           // first rows in the caches
};
template <int MROWS>
__device__ __forceinline__ SeqWork seq_work(const Fp8AttnParams& a, int b) {
  SeqWork w = {};
  w.b = b;
  if (b >= a.batch)
    return w;
  // all loads that do not depend on one another first: a CTA starts with this chain
  const int s0 = __ldg(a.cu_sal + b), s1 = __ldg(a.cu_sal + b + 1);
  const KeyRange kr = keys_of(a, b);
  w.row0 = min(s0, a.num_salient);
  const int n = min(s1, a.num_salient) - w.row0;
  if (n <= 0)
    return w;
  w.rows = n * (a.H / a.Hkv);
  w.k0 = static_cast<int>(kr.k0);
  w.v0 = static_cast<int>(kr.v0);
  w.len = kr.len;
  w.tiles = (w.rows + MROWS - 1) / MROWS;
  return w;
}

// A part of a tile as the scheduler hands it to the other warps.
struct PartInfo {
  int begin, end;              // keys; end < 0: the share is done
  int owner, parts, slot, first;      // several CTAs hold the tile (parts > 1): the first of them, how many, this CTA's slot, it is the first
  int b, hk, row0, rows, t0;   // sequence, key head, the sequence's first listed row, its (row, head) pairs, the tile's first
  int k0, v0, len;             // the sequence's first rows in the caches, its keys
};

// a / b of non-negative numbers; the 64-bit routine only where it is needed.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0)
    return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}
__device__ __forceinline__ int units_of(int2 span) { return max(1, (span.y - span.x + kUnitKeys - 1) / kUnitKeys); }

// Walks over the parts of tiles that a CTA's share of the units consists of, in the order (sequence, tile, key head, keys).
// Uniform over a warp.
//
// Shares are cut at total * i / ctas, but no part of a tile is shorter than kMinPart units: a cut nearer to an end of its
// tile moves there.  Joining the parts of a tile costs a CTA of the few-rows kernel about 7 us, a unit 1 to 2.  With many rows a
// unit takes 5 us and the join is a launch of its own: parts of at least 2 units against 4 take 34.6 us against 43.1 (32 x 601
// keys, 28 heads on 4) and 163 against 166 (4 x 2048 rows of packed documents).
constexpr int kMinPartFew = 4, kMinPartMany = 2;
template <int MROWS>
struct Walk {
  static constexpr int kMinPart = MROWS == kRows ? kMinPartFew : kMinPartMany;
  SeqWork w;
  int64_t total, end;                   // units: of the launch, end of the share before its cut is moved
  int64_t tile_first;                   // first unit of the tile in the launch
  int tile_base;                        // number of the sequence's first tile
  int2 span;                            // keys that rows of the tile see
  int hk, tile, units, first, last;     // the part: units [first, last) of the tile's
  int ctas;                             // shares
  bool begun;

  static __device__ __forceinline__ int moved(int cut, int units) {
    if (cut >= kMinPart && units - cut >= kMinPart)
      return cut;
    return 2 * cut < units ? 0 : units;
  }
  static __device__ __forceinline__ int scan(int x, int lane) {      // sum of the lanes up to this one
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, x, s);
      if (lane >= s)
        x += o;
    }
    return x;
  }
  // Units of a sequence's tiles, for one key head.
  static __device__ __forceinline__ int64_t seq_units(const FewParams& p, const SeqWork& x, int base) {
    if (!p.spans)
      return static_cast<int64_t>(x.tiles) * units_of(make_int2(0, x.len));
    int64_t sum = 0;
    for (int t = 0; t < x.tiles; ++t)
      sum += units_of(__ldg(p.spans + base + t));
    return sum;
  }
  __device__ __forceinline__ void open(const FewParams& p) {
    span = p.spans ? __ldg(p.spans + tile_base + tile) : make_int2(0, w.len);
    units = units_of(span);
  }
  __device__ __forceinline__ void start(const FewParams& p) {
    const int lane = threadIdx.x & 31;
    int64_t sum = 0;
    int all_tiles = 0;
    SeqWork x;
    int x_base = 0;
    int64_t mine = 0;
    for (int base = 0; base < p.a.batch; base += 32) {
      x = seq_work<MROWS>(p.a, base + lane);
      const int upto = scan(x.tiles, lane);
      x_base = all_tiles + upto - x.tiles;
      all_tiles += __shfl_sync(0xffffffffu, upto, 31);
      mine = seq_units(p, x, x_base);
      sum += mine;
    }
#pragma unroll
    for (int s = 16; s; s >>= 1)
      sum += __shfl_xor_sync(0xffffffffu, sum, s);
    total = sum * p.a.Hkv;
    ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), max(static_cast<int64_t>(all_tiles) * p.a.Hkv, total / kMinPart)));
    end = tile_first = 0;
    first = 0;
    begun = false;
    if (static_cast<int>(blockIdx.x) >= ctas)
      return;
    const int64_t at = share(blockIdx.x);
    end = share(blockIdx.x + 1);
    int64_t before = 0;
    all_tiles = 0;
    for (int base = 0;; base += 32) {
      if (p.a.batch > 32) {
        x = seq_work<MROWS>(p.a, base + lane);
        const int upto = scan(x.tiles, lane);
        x_base = all_tiles + upto - x.tiles;
        all_tiles += __shfl_sync(0xffffffffu, upto, 31);
        mine = seq_units(p, x, x_base);
      }
      const int64_t here = mine * p.a.Hkv;
      int64_t upto = here;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, upto, s);
        if (lane >= s)
          upto += o;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > at);
      if (hit) {
        const int src = __ffs(hit) - 1;
        before += __shfl_sync(0xffffffffu, upto - here, src);
        tile_base = __shfl_sync(0xffffffffu, x_base, src);
        w = seq_work<MROWS>(p.a, base + src);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    tile = 0;
    if (!p.spans) {
      const int64_t t = quotient(at - before, static_cast<int64_t>(units_of(make_int2(0, w.len))) * p.a.Hkv);
      tile = static_cast<int>(t);
      open(p);
      tile_first = before + t * units * p.a.Hkv;
    } else {
      tile_first = before;
      for (;; ++tile) {
        open(p);
        if (tile_first + static_cast<int64_t>(units) * p.a.Hkv > at)
          break;
        tile_first += static_cast<int64_t>(units) * p.a.Hkv;
      }
    }
    hk = static_cast<int>(quotient(at - tile_first, units));
    tile_first += static_cast<int64_t>(hk) * units;
    first = moved(static_cast<int>(at - tile_first), units);
  }
  // The next part, false at the end of the share.
  __device__ __forceinline__ bool next(const FewParams& p) {
    if (tile_first >= end)
      return false;
    if (begun || first == units) {
      first = 0;
      tile_first += units;
      if (tile_first >= end)
        return false;
      if (++hk == p.a.Hkv) {
        hk = 0;
        if (++tile == w.tiles) {
          tile = 0;
          do {
            tile_base += w.tiles;
            w = seq_work<MROWS>(p.a, w.b + 1);
          } while (w.tiles == 0);
        }
        open(p);
      }
    }
    begun = true;
    last = tile_first + units <= end ? units : moved(static_cast<int>(end - tile_first), units);
    return last > first;
  }
  // First unit of a share before its cut is moved; CTA that holds the first part of the tile; number of its parts.
  __device__ __forceinline__ int64_t share(int64_t cta) const { return quotient(total * cta, ctas); }
  __device__ __forceinline__ int first_cut() const {
    return static_cast<int>(quotient((tile_first + kMinPart) * ctas + total - 1, total));
  }
  __device__ __forceinline__ int owner() const { return first_cut() - 1; }
  __device__ __forceinline__ int parts() const {
    return static_cast<int>(quotient((tile_first + units - kMinPart + 1) * ctas + total - 1, total)) - first_cut() + 1;
  }
  // What the other warps need to know of the part.
  __device__ __forceinline__ PartInfo info() const {
    const int begin = span.x + first * kUnitKeys;
    PartInfo v = {begin, min(span.y, span.x + last * kUnitKeys), 0, 1, 0, 0, w.b, hk, w.row0, w.rows, tile * MROWS, w.k0, w.v0, w.len};
    if (last - first < units) {
      v.owner = owner();
      v.parts = parts();
      v.first = first == 0 ? 1 : 0;
      v.slot = 2 * static_cast<int>(blockIdx.x) + v.first;
    }
    return v;
  }
};

// One arrival for the warp, after what all of its lanes have done (an arrival per lane is a shared-memory atomic each).
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0)
    mbar_arrive(bar);
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }

__device__ __forceinline__ void group_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(2 + group) : "memory"); }
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Sum of each of N = 8 or 16 values over the lanes of a warp: lane l gets that of value l / (32 / N).
template <int N>
__device__ __forceinline__ float reduce_lanes(const float (&v)[N]) {
  const int lane = threadIdx.x & 31;
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
        x[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
      }
  }
#pragma unroll
  for (int b = 16 / N; b >= 1; b >>= 1)
    x[0] += __shfl_xor_sync(0xffffffffu, x[0], b);
  return x[0];
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

// One step of a product of 8-bit tiles with rows of 128 bytes (128-byte swizzle, groups of 8 rows 1024 bytes apart) at these
// shared-memory addresses.  Only the low words of the descriptors vary: an issue costs few instructions.
__device__ __forceinline__ void umma_tile(uint32_t d_tmem, uint32_t a_addr, uint32_t b_addr, uint32_t idesc, uint32_t accumulate) {
  constexpr uint32_t high = (1024u >> 4) | (1u << 14) | (2u << 29);      // stride, version, swizzle
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"((a_addr >> 4) | (1u << 16)), "r"((b_addr >> 4) | (1u << 16)), "r"(idesc), "r"(accumulate), "n"(high)
      : "memory");
}

// A value that all lanes share, in a register of the uniform datapath: what depends on it alone (loop counters, descriptors)
// stays there, and an MMA issues every 33 cycles (its A operand's shared-memory read) instead of every 90.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }

__device__ __forceinline__ void loaders_sync() { asm volatile("bar.sync 7, 128;" ::: "memory"); }

// Zeros for the rows t0 .. t0 + count - 1 of a sequence's (listed row, head) pairs; one warp.
__device__ __forceinline__ void zero_rows(const Fp8AttnParams& a, const SeqWork& w, int hk, int t0, int count) {
  const int group = a.H / a.Hkv;
  for (int t = t0; t < min(t0 + count, w.rows); ++t) {
    const int i = t / group;
    __nv_bfloat16* dst = a.out + ((static_cast<int64_t>(w.row0) + i) * a.H + hk * group + t - i * group) * kD;
    *reinterpret_cast<uint2*>(dst + (threadIdx.x & 31) * 4) = make_uint2(0u, 0u);
  }
}

// Sixteen elements of a query times `inv` as codes: e4m3, and the rest in e5m2.
__device__ __forceinline__ void split_query(const uint4& x0, const uint4& x1, float inv, uint4& hi, uint4& lo) {
  float y[16];
  bf16x8_to_float(x0, y);
  bf16x8_to_float(x1, y + 8);
  uint32_t h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      z[e] = y[4 * j + e] * inv;
    h[j] = fp8_pack2(z[0], z[1]) | fp8_pack2(z[2], z[3]) << 16;
    const float2 u = fp8_to_float2(h[j] & 0xffffu), v = fp8_to_float2(h[j] >> 16);
    l[j] = fp8_pack2_e5m2(z[0] - u.x, z[1] - u.y) | fp8_pack2_e5m2(z[2] - v.x, z[3] - v.y) << 16;
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

constexpr float kNothing = -1.0e30f;      // maximum of no scores (finite: it takes part in differences)

// Four weights (times 256) as codes and the codes of 16 times what they leave.  By way of half precision (2^-11).
__device__ __forceinline__ void split_weights(const float (&w)[4], uint32_t& hi, uint32_t& lo) {
  uint32_t h[2], l[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 x = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
    h[i] = fp8_pack_half2(*reinterpret_cast<const uint32_t*>(&x));
    const uint32_t back = fp8_to_half2(h[i]);
    const __half2 rest = __hmul2(__hsub2(x, *reinterpret_cast<const __half2*>(&back)), __float2half2_rn(16.f));
    l[i] = fp8_pack_half2(*reinterpret_cast<const uint32_t*>(&rest));
  }
  hi = h[0] | h[1] << 16;
  lo = l[0] | l[1] << 16;
}

// What a tile's rows are to the softmax warps.
struct RowInfo {
  int out;                     // output row, -1: none
  float fix;                   // 1; 0: the row does not exist in q; NaN: the query is not finite
  float slope;                 // times log2(e)
  int pos, lo, hi;             // the row's place in its sequence, the keys that it sees
};

// Joins the parts of a tile that several CTAs hold: every CTA leaves its part in the workspace, the last one to do so adds them
// up in their order (true: for the caller to store).  Rows r0 .. r0 + 7, head dimension kl of a thread.
__device__ __forceinline__ bool join_parts(const FewParams& p, const PartInfo& part, float (&top)[kGroup], float (&l)[kGroup],
                                           float (&o)[kGroup], int r0, int kl, int tid, int* joins) {
  constexpr int kPart = kRows * kD + 2 * kRows;
  float* mine = p.parts + static_cast<int64_t>(part.slot) * kPart;
#pragma unroll
  for (int r = 0; r < kGroup; ++r)
    mine[(r0 + r) * kD + kl] = o[r];
  if (kl == 0) {
#pragma unroll
    for (int r = 0; r < kGroup; ++r) {
      mine[kRows * kD + r0 + r] = top[r];
      mine[kRows * kD + kRows + r0 + r] = l[r];
    }
  }
  const int owner = part.owner, parts = part.parts;
  __threadfence();
  softmax_sync();
  if (tid == 0) {
    open_join(p.tickets + owner, p.launch_id);
    *joins = last_to_join(p.tickets + owner, parts) ? 1 : 0;
  }
  softmax_sync();
  if (!*joins)
    return false;
  __threadfence();
  const float* first = p.parts + (2 * static_cast<int64_t>(owner) + 1) * kPart;
  const float* rest = p.parts + 2 * static_cast<int64_t>(owner) * kPart;
#pragma unroll
  for (int r = 0; r < kGroup; ++r) {
    top[r] = kNothing;
    o[r] = l[r] = 0.f;
  }
  for (int i = 0; i < parts; ++i) {
    const float* src = i == 0 ? first : rest + 2 * static_cast<int64_t>(i) * kPart;
#pragma unroll
    for (int r = 0; r < kGroup; ++r)
      top[r] = fmaxf(top[r], __ldcg(src + kRows * kD + r0 + r));
  }
#pragma unroll 2
  for (int i = 0; i < parts; ++i) {
    const float* src = i == 0 ? first : rest + 2 * static_cast<int64_t>(i) * kPart;
#pragma unroll
    for (int r = 0; r < kGroup; ++r) {
      const float mul = exp2f(__ldcg(src + kRows * kD + r0 + r) - top[r]);
      l[r] += __ldcg(src + kRows * kD + kRows + r0 + r) * mul;
      o[r] += __ldcg(src + (r0 + r) * kD + kl) * mul;
    }
  }
  return true;
}

// The query rows of a tile on their way to shared memory: eight threads a row (the first 256 softmax threads), 16 elements each.
struct QueryLoad {
  uint4 x0, x1;
  int row, head, t;
  __device__ __forceinline__ void index(const Fp8AttnParams& a, const PartInfo& w, int tid) {
    const int group = a.H / a.Hkv;
    row = -1;
    t = w.t0 + (tid >> 3);
    const int i = t / group;
    head = w.hk * group + t - i * group;
    if (t < w.rows)
      row = __ldg(a.idx + w.row0 + i);      // looked at in data(), not while it is on its way
  }
  __device__ __forceinline__ void data(const Fp8AttnParams& a, int tid) {
    row = row >= a.total_q ? -1 : row;
    x0 = x1 = make_uint4(0u, 0u, 0u, 0u);
    if (row >= 0) {
      const uint4* src = reinterpret_cast<const uint4*>(a.q + row * a.ldq + head * kD) + (tid & 7) * 2;
      x0 = __ldg(src);
      x1 = __ldg(src + 1);
    }
  }
  // Codes next to the tile's largest element (an error of 2^-26 of it moves every score of the tile by as little), e4m3 and
  // the e5m2 rest.
  template <bool PLAIN>
  __device__ __forceinline__ void store(const Fp8AttnParams& a, const PartInfo& w, int tid, uint8_t* q_smem, uint32_t* amax, RowInfo* info) {
    float y[16];
    bf16x8_to_float(x0, y);
    bf16x8_to_float(x1, y + 8);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
    m = fp8_amax8(m);
    const bool finite = m < 0x7f800000u;
    {
      const uint32_t top = __reduce_max_sync(0xffffffffu, finite ? m : 0u);
      if ((tid & 31) == 0)
        atomicMax(amax, top);
    }
    asm volatile("bar.sync 6, 256;" ::: "memory");
    const int r = tid >> 3, part = tid & 7;
    const float inv = fp8_inverse(fp8_scale_bits(*amax));
    uint4 hi, lo;
    if (!finite)
      x0 = x1 = make_uint4(0u, 0u, 0u, 0u);
    split_query(x0, x1, inv, hi, lo);
    uint8_t* dst = q_smem + r * kD + ((part ^ (r & 7)) << 4);
    *reinterpret_cast<uint4*>(dst) = hi;
    *reinterpret_cast<uint4*>(dst + kRows * kD) = lo;
    if (part == 0) {
      RowInfo v = {};
      v.out = t < w.rows ? (w.row0 + t / (a.H / a.Hkv)) * a.H + head : -1;
      v.fix = row < 0 ? 0.f : finite ? 1.f : __uint_as_float(0x7fc00000u);
      if (!PLAIN && row >= 0) {
        v.pos = __ldg(a.cu_k + w.b + 1) - __ldg(a.cu_k + w.b) - (__ldg(a.cu_q + w.b + 1) - row);
        v.slope = a.slopes ? __ldg(a.slopes + head) * kLog2e : 0.f;
        v.hi = w.len;
        if (a.ranges) {
          const int2 range = __ldg(a.ranges + row);
          v.lo = range.x;
          v.hi = min(range.y, w.len);
        }
      }
      info[r] = v;
    }
    fence_proxy_async_smem();
  }
};

// The chunks of a CTA's share one after the other, as the producer and the MMA warp walk over them.  Uniform over a warp.
struct Chunks {
  int n, c0, tiles;            // part, first tile of the chunk, tiles of the part
  int begin, end, hk, k0, v0;
  __device__ __forceinline__ int count() const { return min(kChunk, tiles - c0); }
  __device__ __forceinline__ bool open(uint64_t* full, uint64_t* done, const PartInfo* parts, int* abort_flag, int* status) {
    const int slot = n % kParts;
    if (!mbar_wait(&full[slot], (n / kParts) & 1, abort_flag, status, 420))
      return false;
    const PartInfo& w = parts[slot];
    begin = uniform(w.begin);
    end = static_cast<int>(uniform(w.end + 1)) - 1;
    hk = uniform(w.hk);
    k0 = uniform(w.k0);
    v0 = uniform(w.v0);
    warp_arrive(&done[slot]);
    c0 = 0;
    tiles = (end - begin + kUnitKeys - 1) / kUnitKeys;
    return end >= 0;
  }
  __device__ __forceinline__ bool next(uint64_t* full, uint64_t* done, const PartInfo* parts, int* abort_flag, int* status) {
    c0 += kChunk;
    if (c0 < tiles)
      return true;
    ++n;
    return open(full, done, parts, abort_flag, status);
  }
};

template <bool PLAIN>
__global__ void __launch_bounds__(kFewThreads, 1)
fp8_few_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const FewParams p) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  const Fp8AttnParams& a = p.a;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // weights of a chunk: tile i in block i / 2; row = key, 64 bytes at 64 * (i % 2): kRows weights, then kRows remainders
  uint8_t* p_smem = ring + kRing * kTileBytes;
  uint8_t* q_smem = p_smem + kChunk / 2 * kTileBytes;        // two slots of [kRows][128] e4m3, then e5m2
  float* sc_smem = reinterpret_cast<float*>(q_smem + 4 * kQBytes);      // two slots of [kChunk][K, V][128] scales
  __shared__ uint64_t full[kRing], empty[kRing], part_full[kParts], part_done[kParts], q_full[2], s_full[2], s_free[2], p_full, pv_done;
  __shared__ PartInfo s_part[kParts];
  __shared__ uint32_t tmem_slot, s_amax[kParts];
  __shared__ int abort_flag, joins;
  __shared__ RowInfo s_row[2][kRows];
  __shared__ __align__(16) float s_max[4][kRows], s_sum[4][kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kParts; ++i) {
      mbar_init(&part_full[i], 1);
      mbar_init(&part_done[i], kSoftmaxWarps + 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 8);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], kSoftmaxWarps);
    }
    mbar_init(&p_full, kSoftmaxWarps);
    mbar_init(&pv_done, 1);
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
  const uint32_t tmem = tmem_slot;      // S^T of two chunks, then O^T: kRows columns of 256 w, kRows of remainders

  if (warp == kSoftmaxWarps + 2) {
    // ---------------------------------------------------------------- scheduler: the parts of this CTA's share
    Walk<kRows> walk;
    walk.start(p);
    for (int n = 0;;) {
      const bool more = walk.next(p);
      if (more && walk.span.y <= walk.span.x) {      // no keys: zeros
        zero_rows(a, walk.w, walk.hk, walk.tile * kRows, kRows);
        continue;
      }
      const int slot = n % kParts;
      if (n >= kParts && !mbar_wait(&part_done[slot], (n / kParts - 1) & 1, &abort_flag, p.status_word, 400))
        break;
      if (lane == 0) {
        PartInfo v = {};
        v.end = -1;
        if (more)
          v = walk.info();
        s_part[slot] = v;
        s_amax[slot] = 0;
      }
      warp_arrive(&part_full[slot]);
      ++n;
      if (!more)
        break;
    }
  } else if (warp == 0) {
    // ---------------------------------------------------------------- producer: the K tiles of a chunk before the V tiles of the last
    int n = 0;
    auto load = [&](const CUtensorMap* map, const Chunks& c, int row0) {
      for (int i = 0; i < c.count(); ++i, ++n) {
        const int slot = n % kRing, key = c.begin + (c.c0 + i) * kUnitKeys;
        if (n >= kRing)
          mbar_wait(&empty[slot], (n / kRing - 1) & 1, &abort_flag, p.status_word, 401);
        if (elect_one()) {
          const int boxes = min(4, (c.end - key + 31) / 32);      // no box of keys that do not belong to the part
          mbar_arrive_expect_tx(&full[slot], boxes * 32 * kD);
          for (int j = 0; j < boxes; ++j)
            tma_load_2d(ring + slot * kTileBytes + j * 32 * kD, map, &full[slot], c.hk * kD, row0 + key + 32 * j);
        }
        __syncwarp();
      }
    };
    Chunks ahead = {};
    bool more = ahead.open(part_full, part_done, s_part, &abort_flag, p.status_word);
    if (more)
      load(&tmap_k, ahead, ahead.k0);
    while (more) {
      const Chunks now = ahead;
      more = ahead.next(part_full, part_done, s_part, &abort_flag, p.status_word);
      if (more)
        load(&tmap_k, ahead, ahead.k0);
      load(&tmap_v, now, now.v0);
    }
    // a CTA may not end with copies on their way, also when a wait of another warp has given up
    for (int i = max(0, n - kRing); i < n; ++i)
      mbar_wait(&full[i % kRing], (i / kRing) & 1, &abort_flag, p.status_word, 402);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer: the scores of a chunk before the sums of the last
    constexpr uint32_t idesc_hi = umma_idesc_f8(128, kRows, 0, 0, 0, 0), idesc_lo = umma_idesc_f8(128, kRows, 0, 1, 0, 0);
    constexpr uint32_t idesc_pv = umma_idesc_f8(128, 2 * kRows, 0, 0, 1, 1);
    const uint32_t ring_addr = smem_u32(ring), p_addr = smem_u32(p_smem), t_s = uniform(tmem), t_o = t_s + 2 * kChunk * kRows;
    int n = 0, n_s = 0, n_p = 0;
    auto scores = [&](const Chunks& c) {
      const int buf = n_s & 1;
      if (c.c0 == 0)
        mbar_wait(&q_full[c.n & 1], (c.n >> 1) & 1, &abort_flag, p.status_word, 403);
      if (n_s >= 2)
        mbar_wait(&s_free[buf], ((n_s >> 1) - 1) & 1, &abort_flag, p.status_word, 404);
      const uint32_t q_addr = smem_u32(q_smem) + (c.n & 1) * 2 * kQBytes;
      const int nt = c.count();
      for (int i = 0; i < nt; ++i, ++n) {
        const int slot = n % kRing;
        mbar_wait(&full[slot], (n / kRing) & 1, &abort_flag, p.status_word, 405);
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t k_addr = ring_addr + slot * kTileBytes, d = t_s + (buf * kChunk + i) * kRows;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {      // 32 head dimensions = 32 bytes a step
            umma_tile(d, k_addr + 32 * kk, q_addr + 32 * kk, idesc_hi, kk != 0 ? 1u : 0u);
            umma_tile(d, k_addr + 32 * kk, q_addr + kQBytes + 32 * kk, idesc_lo, 1u);
          }
          umma_commit(&empty[slot]);
          if (i == nt - 1)
            umma_commit(&s_full[buf]);
        }
        __syncwarp();
      }
      ++n_s;
    };
    Chunks ahead = {};
    bool more = ahead.open(part_full, part_done, s_part, &abort_flag, p.status_word);
    if (more)
      scores(ahead);
    while (more) {
      const Chunks now = ahead;
      more = ahead.next(part_full, part_done, s_part, &abort_flag, p.status_word);
      if (more)
        scores(ahead);
      const int nt = now.count();
      mbar_wait(&p_full, n_p & 1, &abort_flag, p.status_word, 407);
      ++n_p;
      for (int i = 0; i < nt; ++i, ++n) {
        const int slot = n % kRing;
        mbar_wait(&full[slot], (n / kRing) & 1, &abort_flag, p.status_word, 406);
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t v_addr = ring_addr + slot * kTileBytes, w_addr = p_addr + (i >> 1) * kTileBytes + (i & 1) * 64;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)        // 32 keys = 32 rows of 128 bytes a step
            umma_tile(t_o, v_addr + kk * 4096, w_addr + kk * 4096, idesc_pv, (now.c0 | i | kk) != 0 ? 1u : 0u);
          umma_commit(&empty[slot]);
          if (i == nt - 1)
            umma_commit(&pv_done);
        }
        __syncwarp();
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax over the keys, epilogue
    const int rg = (warp - 2) >> 2;                // rows kGroup * rg ..
    const int quarter = warp & 3;                  // tensor-memory lanes: keys (head dimensions) 32 * quarter ..
    const int tid = threadIdx.x - 64;
    const int kl = quarter * 32 + lane;            // key of a tile, or head dimension
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_o = t_lane + 2 * kChunk * kRows;
    const int r0 = rg * kGroup;
    const bool stages = warp < 10;                 // takes part in staging the queries
    const float key_mul = a.scale * (PLAIN ? kLog2e : 1.f);
    uint8_t* p_dst = p_smem + kl * kD + (rg & 1) * 8;

    // Scales of the keys of a chunk, copied ahead of their use: K's by the first half of the threads, V's by the second.  The
    // heads of a key lie side by side: CTAs that work on them at the same time start at different tiles.
    auto request_scales = [&](const PartInfo& w, int key, int slot) {
      const bool of_v = tid >= 256;
      const float* src = (of_v ? a.v_scales + static_cast<int64_t>(w.v0) * a.Hkv : a.k_scales + static_cast<int64_t>(w.k0) * a.Hkv) + w.hk;
      float* dst = sc_smem + slot * kChunk * 2 * kUnitKeys + (of_v ? kUnitKeys : 0) + (tid & 127);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = (2 * j + ((tid >> 7) & 1) + w.hk) & (kChunk - 1), at = key + i * kUnitKeys + (tid & 127);
        if (at < w.end)
          cp_async4(dst + i * 2 * kUnitKeys, src + static_cast<int64_t>(at) * a.Hkv);
      }
      cp_async_commit();
    };
    auto wait_part = [&](int n) {
      return mbar_wait(&part_full[n % kParts], (n / kParts) & 1, &abort_flag, p.status_word, 415) && s_part[n % kParts].end >= 0;
    };
    auto stage = [&](int n, QueryLoad& ql) {
      if (stages) {
        ql.template store<PLAIN>(a, s_part[n % kParts], tid, q_smem + (n & 1) * 2 * kQBytes, &s_amax[n % kParts], s_row[n & 1]);
        warp_arrive(&q_full[n & 1]);
      }
    };

    QueryLoad ql;
    int n_chunk = 0, ring_at = 0;
    bool more = wait_part(0), after = false;       // whether the part at hand and the one after it exist
    if (more) {
      request_scales(s_part[0], s_part[0].begin, 0);
      if (stages) {
        ql.index(a, s_part[0], tid);
        ql.data(a, tid);
      }
      stage(0, ql);
      after = wait_part(1);
      if (after && stages) {
        ql.index(a, s_part[1], tid);
        ql.data(a, tid);
      }
      cp_async_wait_all();
      softmax_sync();
      ring_at = min(kChunk, (s_part[0].end - s_part[0].begin + kUnitKeys - 1) / kUnitKeys);
    }
    for (int n = 0; more; ++n) {
      const PartInfo& part = s_part[n % kParts];
      const RowInfo* rows = &s_row[n & 1][r0];
      const int end = part.end, tiles = (end - part.begin + kUnitKeys - 1) / kUnitKeys;
      const bool alive = rows[0].out >= 0;         // rows are filled from the first on
      bool then = false;                           // whether the part after the next exists
      float top[kGroup], l[kGroup];
#pragma unroll
      for (int r = 0; r < kGroup; ++r) {
        top[r] = kNothing;
        l[r] = 0.f;
      }
      for (int c0 = 0; c0 < tiles; c0 += kChunk, ++n_chunk) {
        const int nt = min(kChunk, tiles - c0), buf = n_chunk & 1;
        const bool last = c0 + kChunk >= tiles;
        const int key0 = part.begin + c0 * kUnitKeys + kl;
        float kk[kChunk], ex[kChunk];
        {
          const float* sc = sc_smem + buf * kChunk * 2 * kUnitKeys + kl;
          const float mul = key_mul * __uint_as_float(fp8_scale_bits(s_amax[n % kParts]));
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            kk[i] = sc[i * 2 * kUnitKeys] * mul;
            ex[i] = value_exponent(sc[(i * 2 + 1) * kUnitKeys]);
          }
        }
        // products of the chunk; tensor memory is free for the next one
        mbar_wait(&s_full[buf], (n_chunk >> 1) & 1, &abort_flag, p.status_word, 409);
        tc_fence_after_sync();
        uint32_t s[kChunk][kGroup];
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
          if (i < nt)
            tmem_ld_32x8(t_lane + (buf * kChunk + i) * kRows + r0, s[i]);
        tmem_ld_wait();
        tc_fence_before_sync();
        warp_arrive(&s_free[buf]);
        // what the next chunk needs
        int next_tiles = 0;
        if (!last) {
          request_scales(part, part.begin + (c0 + kChunk) * kUnitKeys, buf ^ 1);
          next_tiles = min(kChunk, tiles - c0 - kChunk);
        } else if (after) {
          stage(n + 1, ql);
          const PartInfo& w = s_part[(n + 1) % kParts];
          request_scales(w, w.begin, buf ^ 1);
          next_tiles = min(kChunk, (w.end - w.begin + kUnitKeys - 1) / kUnitKeys);
          then = wait_part(n + 2);
          if (then && stages)
            ql.index(a, s_part[(n + 2) % kParts], tid);
        }
        const int v_at = ring_at + next_tiles;      // the chunk's V tiles in the order of the ring
        ring_at = v_at + nt;

        float mx[kGroup];
#pragma unroll
        for (int r = 0; r < kGroup; ++r)
          mx[r] = top[r];
        if (alive) {
          // scores (times log2 e, plus the exponents of the values' scales) and their maxima
          if (PLAIN) {
#pragma unroll
            for (int i = 0; i < kChunk; ++i)
              if (key0 + i * kUnitKeys < end) {
#pragma unroll
                for (int r = 0; r < kGroup; ++r) {
                  const float t = fmaf(__uint_as_float(s[i][r]), kk[i], ex[i]);
                  s[i][r] = __float_as_uint(t);
                  mx[r] = fmaxf(mx[r], t);
                }
              }
          } else {
#pragma unroll
            for (int i = 0; i < kChunk; ++i)
#pragma unroll
              for (int r = 0; r < kGroup; ++r)
                s[i][r] = __float_as_uint(__uint_as_float(s[i][r]) * kk[i]);
            if (a.cap > 0.f) {
              const float to = 2.f * kLog2e / a.cap;
#pragma unroll
              for (int i = 0; i < kChunk; ++i)
#pragma unroll
                for (int r = 0; r < kGroup; ++r)
                  s[i][r] = __float_as_uint(capped(__uint_as_float(s[i][r]) * to, a.cap));
            }
#pragma unroll
            for (int r = 0; r < kGroup; ++r) {
              const float slope = rows[r].slope;
              const int pos = rows[r].pos, lo = rows[r].lo, hi = min(rows[r].hi, end);
#pragma unroll
              for (int i = 0; i < kChunk; ++i) {
                const int at = key0 + i * kUnitKeys;
                float t = fmaf(__uint_as_float(s[i][r]), kLog2e, ex[i]) - slope * static_cast<float>(abs(pos - at));
                t = at >= lo && at < hi ? t : -INFINITY;
                s[i][r] = __float_as_uint(t);
                mx[r] = fmaxf(mx[r], t);
              }
            }
          }
#pragma unroll
          for (int r = 0; r < kGroup; ++r)
            mx[r] = warp_max(mx[r]);
          if (lane == 0) {
#pragma unroll
            for (int r = 0; r < kGroup; r += 4)
              *reinterpret_cast<float4*>(&s_max[quarter][r0 + r]) = make_float4(mx[r], mx[r + 1], mx[r + 2], mx[r + 3]);
          }
          group_sync(rg);
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            float x[kGroup];
            lds_row(x, s_max[q4] + r0);
#pragma unroll
            for (int r = 0; r < kGroup; ++r)
              mx[r] = fmaxf(mx[r], x[r]);
          }
        }
        // the weights of the last chunk have been taken; the sums are rescaled where a maximum has grown
        if (n_chunk > 0)
          mbar_wait(&pv_done, (n_chunk - 1) & 1, &abort_flag, p.status_word, 410);
        if (alive) {
          bool grown = false;
#pragma unroll
          for (int r = 0; r < kGroup; ++r)
            grown = grown || mx[r] > top[r];
          if (c0 > 0 && grown) {      // the same rows in all four quarters
            float old[kGroup];
#pragma unroll
            for (int r = 0; r < kGroup; ++r) {
              old[r] = exp2f(top[r] - mx[r]);
              l[r] *= old[r];
            }
            tc_fence_after_sync();
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t o[kGroup];
              tmem_ld_32x8(t_o + j * kRows + r0, o);
              tmem_ld_wait();
#pragma unroll
              for (int r = 0; r < kGroup; ++r)
                o[r] = __float_as_uint(__uint_as_float(o[r]) * old[r]);
              tmem_st_32x8(t_o + j * kRows + r0, o);
            }
            tmem_st_wait();
          }
#pragma unroll
          for (int r = 0; r < kGroup; ++r) {
            top[r] = mx[r];
            mx[r] = 8.f - mx[r];      // weights are taken times 256
          }
#pragma unroll
          for (int i = 0; i < kChunk; ++i)
            if (i < nt) {
              uint32_t hi[2] = {0u, 0u}, lo[2] = {0u, 0u};
              if (key0 + i * kUnitKeys < end) {
                // the weight of a NaN is a NaN where its key is seen, else zero
                const float inv = ex[i] == ex[i] ? exp2f(-ex[i]) : 1.f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  float w4[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    w4[e] = exp2f(__uint_as_float(s[i][4 * j + e]) + mx[4 * j + e]);
                    l[4 * j + e] = fmaf(w4[e], inv, l[4 * j + e]);
                  }
                  split_weights(w4, hi[j], lo[j]);
                }
              }
              uint8_t* dst = p_dst + (i >> 1) * kTileBytes;
              *reinterpret_cast<uint2*>(dst + (((4 * (i & 1) + (rg >> 1)) ^ (kl & 7)) << 4)) = make_uint2(hi[0], hi[1]);
              *reinterpret_cast<uint2*>(dst + (((4 * (i & 1) + 2 + (rg >> 1)) ^ (kl & 7)) << 4)) = make_uint2(lo[0], lo[1]);
            }
        }
        if (last && end - (key0 - kl) < nt * kUnitKeys && rg == 0) {
          // rows behind the last key may hold any byte, a NaN times a weight of zero among them
          const int use = v_at + nt - 1;
          mbar_wait(&full[use % kRing], (use / kRing) & 1, &abort_flag, p.status_word, 412);
          if (key0 + (nt - 1) * kUnitKeys >= end) {
            uint4* v = reinterpret_cast<uint4*>(ring + (use % kRing) * kTileBytes + kl * kD);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              v[j] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        tc_fence_before_sync();
        fence_proxy_async_smem();
        warp_arrive(&p_full);
        if (!last) {
          cp_async_wait_all();
          softmax_sync();      // everybody's scales of the next chunk are there
        }
      }

      // ---------------------------------------------------------------- thread = head dimension kl of kGroup rows
      if (then && stages)
        ql.data(a, tid);
      {
        const float v = reduce_lanes<kGroup>(l);
        if (lane % (32 / kGroup) == 0)
          s_sum[quarter][r0 + lane / (32 / kGroup)] = v;
      }
      int dst[kGroup];
      float fix[kGroup];
#pragma unroll
      for (int r = 0; r < kGroup; ++r) {
        dst[r] = rows[r].out;
        fix[r] = rows[r].fix;
      }
      const PartInfo joined = part;
      cp_async_wait_all();
      softmax_sync();          // the sums and the next part's scales and rows are there; this part's descriptions are not read again
      warp_arrive(&part_done[n % kParts]);
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        float x[kGroup];
        lds_row(x, s_sum[q4] + r0);
#pragma unroll
        for (int r = 0; r < kGroup; ++r)
          l[r] = q4 == 0 ? x[r] : l[r] + x[r];
      }
      mbar_wait(&pv_done, (n_chunk - 1) & 1, &abort_flag, p.status_word, 413);
      tc_fence_after_sync();
      float o[kGroup];
      {
        uint32_t u[kGroup], v[kGroup];
        tmem_ld_32x8(t_o + r0, u);
        tmem_ld_32x8(t_o + kRows + r0, v);
        tmem_ld_wait();
#pragma unroll
        for (int r = 0; r < kGroup; ++r)
          o[r] = fmaf(__uint_as_float(v[r]), 0.0625f, __uint_as_float(u[r]));
      }
      tc_fence_before_sync();
      if (joined.parts == 1 || join_parts(p, joined, top, l, o, r0, kl, tid, &joins)) {
#pragma unroll
        for (int r = 0; r < kGroup; ++r)
          if (dst[r] >= 0)
            a.out[static_cast<int64_t>(dst[r]) * kD + kl] =
                __float2bfloat16_rn(l[r] == 0.f || fix[r] == 0.f ? 0.f : o[r] * __fdividef(fix[r], l[r]));
      }
      more = after;
      after = then;
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ----------------------------------------------------------------------------------------------
// Many rows per sequence: bound by the exponentials and the instructions around them (a tile of 128 rows x 128 keys takes the
// tensor cores 950 cycles, its exponentials 1024).
//
// Tiles of 128 (listed row, query head) pairs, rows in the M = 128 of the products:
//   S = Q K^T    A: the queries as e4m3 + e5m2 (two products into one accumulator), B: the K tile as loaded (K-major)
//   O = P V      A: the weights as e4m3 + e5m2, B: the V tile as loaded (MN-major)
// Thread = row in four softmax warps.  A weight is 64 * 2^(t - reference); the reference follows the maximum in steps, so that the
// sums are rescaled only where a score lies more than 2.8 (log2) above it.  A weight is off by 2^-7 of itself or by 2^-23 of the
// largest.  Scores and weights share 128 columns of tensor memory (32 keys' weights, e4m3 then e5m2, lie in the first 16 of their
// scores' 32 columns), so the steps of one tile follow one another; two CTAs per SM, each with parts of its own, fill each other's
// waits, the ends of parts among them.  Four loader warps stage the queries of the next part and the scales of the next tiles.
// ----------------------------------------------------------------------------------------------
constexpr int kManyRows = 128;
constexpr int kManyRing = 4;                                 // slots of one K or V tile
constexpr int kScaleSlots = 2;                               // tiles whose scales are staged ahead
constexpr int kManyWarps = 4, kManyThreads = 32 * (3 + kManyWarps + 4);
constexpr int kManyCtas = 2;                                 // per SM
constexpr uint32_t kManyTmemCols = 256;
constexpr uint32_t kStageBytes = 32 * 64;                    // of a softmax warp: 32 head dimensions of its rows
constexpr uint32_t kManyQBytes = kManyRows * kD;             // e4m3 or e5m2 part of the queries of a tile
constexpr uint32_t kManySmem = kManyRing * kTileBytes + 2 * kManyQBytes + kManyWarps * kStageBytes +
                               kScaleSlots * 3 * kUnitKeys * sizeof(float) + 1024;
constexpr float kWeightLog2 = 6.f;                           // the reference's weight: 2^6
constexpr float kHeadroom = 2.8f;                            // 2^(6 + 2.8) < 448

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Pairs of floats in one instruction.
__device__ __forceinline__ float2 get2(const float* x) { return make_float2(x[0], x[1]); }
__device__ __forceinline__ void put2(float* x, float2 v) {
  x[0] = v.x;
  x[1] = v.y;
}
__device__ __forceinline__ uint64_t bits2(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 floats2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return floats2(r);
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return floats2(r);
}
// The lowest n bits.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// Four weights as codes, and what they leave in e5m2.  By way of half precision (2^-11).
__device__ __forceinline__ void split_weights_e5m2(float2 a, float2 b, uint32_t& hi, uint32_t& lo) {
  const __half2 x = __floats2half2_rn(a.x, a.y), y = __floats2half2_rn(b.x, b.y);
  const uint32_t h0 = fp8_pack_half2(*reinterpret_cast<const uint32_t*>(&x)), h1 = fp8_pack_half2(*reinterpret_cast<const uint32_t*>(&y));
  const uint32_t u = fp8_to_half2(h0), v = fp8_to_half2(h1);
  const __half2 r = __hsub2(x, *reinterpret_cast<const __half2*>(&u)), s = __hsub2(y, *reinterpret_cast<const __half2*>(&v));
  hi = __byte_perm(h0, h1, 0x5410);
  lo = __byte_perm(fp8_pack_half2_e5m2(*reinterpret_cast<const uint32_t*>(&r)), fp8_pack_half2_e5m2(*reinterpret_cast<const uint32_t*>(&s)), 0x5410);
}

// A part in the workspace: [dimension][row] sums, [row] references, sums of weights; of a first part also output rows and `fix`.
constexpr int kManyPart = kManyRows * (kD + 4);

// One step of a product whose A operand, 32 codes of a row in 8 columns, lies in tensor memory.
__device__ __forceinline__ void umma_tile_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_addr, uint32_t idesc, uint32_t accumulate) {
  constexpr uint32_t high = (1024u >> 4) | (1u << 14) | (2u << 29);      // as umma_tile
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], b, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"((b_addr >> 4) | (1u << 16)), "r"(idesc), "r"(accumulate), "n"(high)
      : "memory");
}

// CAP, BIAS: scores capped by a tanh, biased by their distance.
template <bool CAP, bool BIAS>
__global__ void __launch_bounds__(kManyThreads, kManyCtas)
fp8_many_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const FewParams p) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  const Fp8AttnParams& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = ring + kManyRing * kTileBytes;           // [128 rows][128] e4m3, then e5m2
  uint8_t* stage = q_smem + 2 * kManyQBytes;
  float* sc_smem = reinterpret_cast<float*>(stage + kManyWarps * kStageBytes);      // per tile: K scale * factors, V exponent, 1 / V scale
  __shared__ uint64_t full[kManyRing], empty[kManyRing], part_full[kParts], part_done[kParts], q_full, q_free, s_full, p_full, pv_done, o_free,
      sc_full[kScaleSlots], sc_free[kScaleSlots];
  __shared__ PartInfo s_part[kParts];
  __shared__ uint32_t tmem_slot, s_amax[2];
  __shared__ int abort_flag;
  __shared__ RowInfo s_row[kManyRows];
  __shared__ int64_t s_src[kManyRows];
  __shared__ uint32_t s_bad[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kManyRing; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kParts; ++i) {
      mbar_init(&part_full[i], 1);
      mbar_init(&part_done[i], kManyWarps + 2 + 4);
    }
    for (int i = 0; i < kScaleSlots; ++i) {
      mbar_init(&sc_full[i], 4);
      mbar_init(&sc_free[i], kManyWarps);
    }
    mbar_init(&q_full, 4);
    mbar_init(&q_free, kManyWarps);
    mbar_init(&s_full, 1);
    mbar_init(&p_full, kManyWarps);
    mbar_init(&pv_done, 1);
    mbar_init(&o_free, kManyWarps);
    fence_mbar_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kManyTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;      // scores and weights: columns 0 .. 127, sums: 128 .. 255
  const int group = a.H / a.Hkv;

  if (warp == 2) {
    // ---------------------------------------------------------------- scheduler
    Walk<kManyRows> walk;
    walk.start(p);
    for (int n = 0;;) {
      const bool more = walk.next(p);
      const int slot = n % kParts;
      if (n >= kParts && !mbar_wait(&part_done[slot], (n / kParts - 1) & 1, &abort_flag, p.status_word, 500))
        break;
      if (lane == 0) {
        PartInfo v = {};
        v.end = -1;
        if (more)
          v = walk.info();
        s_part[slot] = v;
      }
      warp_arrive(&part_full[slot]);
      ++n;
      if (!more)
        break;
    }
  } else if (warp == 0) {
    // ---------------------------------------------------------------- producer: K and V in turn
    int n = 0;
    auto load = [&](const CUtensorMap* map, int row, int left, int x) {
      const int slot = n % kManyRing;
      if (n >= kManyRing)
        mbar_wait(&empty[slot], (n / kManyRing - 1) & 1, &abort_flag, p.status_word, 501);
      if (elect_one()) {
        const int boxes = min(4, (left + 31) / 32);      // no box of keys that do not belong to the part
        mbar_arrive_expect_tx(&full[slot], boxes * 32 * kD);
        for (int j = 0; j < boxes; ++j)
          tma_load_2d(ring + slot * kTileBytes + j * 32 * kD, map, &full[slot], x, row + 32 * j);
      }
      __syncwarp();
      ++n;
    };
    Chunks c = {};
    for (bool more = c.open(part_full, part_done, s_part, &abort_flag, p.status_word); more;) {
      for (int key = c.begin; key < c.end; key += kUnitKeys) {
        load(&tmap_k, c.k0 + key, c.end - key, c.hk * kD);
        load(&tmap_v, c.v0 + key, c.end - key, c.hk * kD);
      }
      ++c.n;
      more = c.open(part_full, part_done, s_part, &abort_flag, p.status_word);
    }
    // a CTA may not end with copies on their way, also when a wait of another warp has given up
    for (int i = max(0, n - kManyRing); i < n; ++i)
      mbar_wait(&full[i % kManyRing], (i / kManyRing) & 1, &abort_flag, p.status_word, 502);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc_hi = umma_idesc_f8(128, 128, 0, 0, 0, 0), idesc_lo = umma_idesc_f8(128, 128, 1, 0, 0, 0);
    constexpr uint32_t idesc_pv = umma_idesc_f8(128, 128, 0, 0, 0, 1), idesc_pv_lo = umma_idesc_f8(128, 128, 1, 0, 0, 1);
    const uint32_t ring_addr = smem_u32(ring), q_addr = smem_u32(q_smem), t_s = uniform(tmem), t_o = t_s + 128;
    int g = 0, live = 0;      // tiles, parts that have some
    Chunks c = {};
    for (bool more = c.open(part_full, part_done, s_part, &abort_flag, p.status_word); more;) {
      if (c.tiles)
        mbar_wait(&q_full, live & 1, &abort_flag, p.status_word, 503);
      for (int i = 0; i < c.tiles; ++i, ++g) {
        const int ks = 2 * g % kManyRing, vs = ks + 1;
        const uint32_t parity = (2 * g / kManyRing) & 1;
        mbar_wait(&full[ks], parity, &abort_flag, p.status_word, 505);
        if (g)
          mbar_wait(&pv_done, (g - 1) & 1, &abort_flag, p.status_word, 504);      // the weights have been taken: their columns are free
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t k_addr = ring_addr + ks * kTileBytes;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {      // 32 head dimensions = 32 bytes a step
            umma_tile(t_s, q_addr + 32 * kk, k_addr + 32 * kk, idesc_hi, kk != 0 ? 1u : 0u);
            umma_tile(t_s, q_addr + kManyQBytes + 32 * kk, k_addr + 32 * kk, idesc_lo, 1u);
          }
          umma_commit(&empty[ks]);
          umma_commit(&s_full);
        }
        __syncwarp();
        mbar_wait(&full[vs], parity, &abort_flag, p.status_word, 506);
        if (i == 0 && live > 0)
          mbar_wait(&o_free, (live - 1) & 1, &abort_flag, p.status_word, 508);
        mbar_wait(&p_full, g & 1, &abort_flag, p.status_word, 507);
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t v_addr = ring_addr + vs * kTileBytes;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {      // 32 keys: 8 columns of weights, 32 rows of V
            umma_tile_ts(t_o, t_s + 32 * kk, v_addr + kk * 4096, idesc_pv, i == 0 && kk == 0 ? 0u : 1u);
            umma_tile_ts(t_o, t_s + 32 * kk + 8, v_addr + kk * 4096, idesc_pv_lo, 1u);
          }
          umma_commit(&empty[vs]);
          umma_commit(&pv_done);
        }
        __syncwarp();
      }
      live += c.tiles ? 1 : 0;
      ++c.n;
      more = c.open(part_full, part_done, s_part, &abort_flag, p.status_word);
    }
  } else if (warp >= 3 + kManyWarps) {
    // ---------------------------------------------------------------- loaders: queries of a part, scales of its tiles
    const int tid = threadIdx.x - 32 * (3 + kManyWarps);
    int n_sc = 0, live = 0;
    for (int n = 0;; ++n) {
      const int slot = n % kParts, qb = live & 1;
      if (!mbar_wait(&part_full[slot], (n / kParts) & 1, &abort_flag, p.status_word, 510))
        break;
      const PartInfo w = s_part[slot];
      loaders_sync();
      warp_arrive(&part_done[slot]);
      if (w.end < 0)
        break;
      // thread = row: where its query lies, what the softmax warps need to know of it
      const int t = w.t0 + tid, i = t / group, head = w.hk * group + t - i * group;
      RowInfo v = {};
      v.out = -1;
      int64_t src = -1;
      if (t < w.rows) {
        v.out = (w.row0 + i) * a.H + head;
        const int at = __ldg(a.idx + w.row0 + i);
        if (at >= 0 && at < a.total_q) {
          src = at * a.ldq + head * kD;
          v.fix = 1.f;
          v.hi = w.len;
          v.pos = __ldg(a.cu_k + w.b + 1) - __ldg(a.cu_k + w.b) - (__ldg(a.cu_q + w.b + 1) - at);
          v.slope = BIAS ? __ldg(a.slopes + head) * kLog2e : 0.f;
          if (a.ranges) {
            const int2 range = __ldg(a.ranges + at);
            v.lo = range.x;
            v.hi = min(range.y, w.len);
          }
        }
      }
      if (w.end == w.begin) {      // no keys: zeros
        s_src[tid] = v.out;
        loaders_sync();
#pragma unroll 1
        for (int r = tid >> 4; r < kManyRows; r += 8)
          if (s_src[r] >= 0)
            *reinterpret_cast<uint4*>(a.out + s_src[r] * kD + (tid & 15) * 8) = make_uint4(0u, 0u, 0u, 0u);
        loaders_sync();
        continue;
      }
      s_src[tid] = src;
      if (tid == 0)
        s_amax[qb] = 0;
      if (tid < 4)
        s_bad[tid] = 0;
      loaders_sync();
      // queries: eight threads a row, 16 rows at a time, four times 16 in flight; first the largest element, then (from L1) the
      // codes.  (Loops: straight-line code for 128 rows that runs once a part costs more in instruction fetches than it saves.)
      uint4 x0[4], x1[4];
      auto fetch = [&](int h) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int64_t from = s_src[64 * h + 16 * k + (tid >> 3)];
          x0[k] = x1[k] = make_uint4(0u, 0u, 0u, 0u);
          if (from >= 0) {
            const uint4* q = reinterpret_cast<const uint4*>(a.q + from) + (tid & 7) * 2;
            x0[k] = __ldg(q);
            x1[k] = __ldg(q + 1);
          }
        }
      };
      uint32_t top = 0;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        fetch(h);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 64 * h + 16 * k + (tid >> 3);
          const uint32_t m = fp8_amax8(max(bf16x8_amax(x0[k]), bf16x8_amax(x1[k])));
          if (m < 0x7f800000u)
            top = max(top, m);
          else if ((tid & 7) == 0)
            atomicOr(&s_bad[r >> 5], 1u << (r & 31));
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0)
        atomicMax(&s_amax[qb], top);
      loaders_sync();
      const uint32_t scale = fp8_scale_bits(s_amax[qb]);
      const float inv = fp8_inverse(scale);
      if (live > 0)
        mbar_wait(&q_free, (live - 1) & 1, &abort_flag, p.status_word, 511);
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        fetch(h);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 64 * h + 16 * k + (tid >> 3), part = tid & 7;
          if (s_bad[r >> 5] >> (r & 31) & 1)
            x0[k] = x1[k] = make_uint4(0u, 0u, 0u, 0u);
          uint4 hi, lo;
          split_query(x0[k], x1[k], inv, hi, lo);
          uint8_t* dst = q_smem + r * kD + ((part ^ (r & 7)) << 4);
          *reinterpret_cast<uint4*>(dst) = hi;
          *reinterpret_cast<uint4*>(dst + kManyQBytes) = lo;
        }
      }
      if (s_bad[tid >> 5] >> (tid & 31) & 1)
        v.fix = __uint_as_float(0x7fc00000u);
      s_row[tid] = v;
      fence_proxy_async_smem();
      loaders_sync();
      warp_arrive(&q_full);
      ++live;
      // scales: thread = key, four tiles' loads at a time
      // scores come out times log2(e), or as twice the argument of the tanh that caps them
      const float mul = a.scale * __uint_as_float(scale) * kLog2e * (CAP ? 2.f / a.cap : 1.f);
      const float* ks = a.k_scales + static_cast<int64_t>(w.k0) * a.Hkv + w.hk;
      const float* vs = a.v_scales + static_cast<int64_t>(w.v0) * a.Hkv + w.hk;
      for (int key = w.begin + tid; key - tid < w.end; key += 4 * kUnitKeys) {
        float x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = key + i * kUnitKeys;
          x[i] = y[i] = 1.f;
          if (at < w.end) {
            x[i] = __ldg(ks + static_cast<int64_t>(at) * a.Hkv);
            y[i] = __ldg(vs + static_cast<int64_t>(at) * a.Hkv);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key - tid + i * kUnitKeys < w.end) {
            const int sl = n_sc % kScaleSlots;
            if (n_sc >= kScaleSlots)
              mbar_wait(&sc_free[sl], (n_sc / kScaleSlots - 1) & 1, &abort_flag, p.status_word, 512);
            const float ex = value_exponent(y[i]);
            float* dst = sc_smem + sl * 3 * kUnitKeys + tid;
            dst[0] = x[i] * mul;
            dst[kUnitKeys] = ex;
            dst[2 * kUnitKeys] = ex == ex ? exp2f(-ex) : 1.f;      // the weight of a NaN is a NaN where its key is seen, else zero
            warp_arrive(&sc_full[sl]);
            ++n_sc;
          }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax: thread = row
    const int quarter = warp & 3;
    const int tid = threadIdx.x - 96;
    const int row = quarter * 32 + lane;
    const uint32_t t_s = tmem + (static_cast<uint32_t>(quarter * 32) << 16), t_o = t_s + 128;
    uint8_t* out_stage = stage + (warp - 3) * kStageBytes;
    int g = 0;                        // tiles so far
    bool owns = false;                // the first part of a tile that goes on in other CTAs
    int live = 0;
    for (int n = 0;; ++n) {
      if (!mbar_wait(&part_full[n % kParts], (n / kParts) & 1, &abort_flag, p.status_word, 515))
        break;
      const PartInfo& part = s_part[n % kParts];
      const int begin = part.begin, end = part.end;
      const bool alive = part.t0 + quarter * 32 < part.rows;
      const int joined_slot = part.slot, joined_parts = part.parts;
      const bool joined_first = part.first != 0;
      if (end <= begin) {
        warp_arrive(&part_done[n % kParts]);
        if (end < 0)
          break;
        continue;
      }
      mbar_wait(&q_full, live & 1, &abort_flag, p.status_word, 516);
      const RowInfo me = s_row[row];
      warp_arrive(&part_done[n % kParts]);
      ++live;
      float ref = kNothing, l = 0.f;
      for (int key0 = begin; key0 < end; key0 += kUnitKeys, ++g) {
        const int sl = g % kScaleSlots;
        const float* sc = sc_smem + sl * 3 * kUnitKeys;
        mbar_wait(&sc_full[sl], (g / kScaleSlots) & 1, &abort_flag, p.status_word, 518);
        mbar_wait(&s_full, g & 1, &abort_flag, p.status_word, 519);      // and with it the product before
        tc_fence_after_sync();
        bool grown = false;
        float old = 1.f;
        if (alive) {
          // scores (times log2 e, plus the exponents of the values' scales), in place of the products, and their maximum
          float mx = kNothing;
          const int lo = me.lo - key0, hi = min(me.hi, end) - key0;
          const float away = static_cast<float>(me.pos - key0);
          uint32_t s[2][16];
          tmem_ld_32x16(t_s, s[0]);
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const uint32_t seen = below(hi - c * 32) & ~below(lo - c * 32);      // of 32 keys
            const bool cut = __any_sync(0xffffffffu, me.out >= 0 && seen != 0xffffffffu);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              tmem_ld_wait();
              if (h == 0 || c < 3)
                tmem_ld_32x16(t_s + c * 32 + (h + 1) * 16, s[h ^ 1]);
              float* t = reinterpret_cast<float*>(s[h]);
              const float d = away - static_cast<float>(c * 32 + h * 16);
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                const float4 kk = *reinterpret_cast<const float4*>(sc + c * 32 + h * 16 + j);
                const float4 ex = *reinterpret_cast<const float4*>(sc + kUnitKeys + c * 32 + h * 16 + j);
                if (!CAP) {
                  put2(t + j, ffma2(get2(t + j), make_float2(kk.x, kk.y), make_float2(ex.x, ex.y)));
                  put2(t + j + 2, ffma2(get2(t + j + 2), make_float2(kk.z, kk.w), make_float2(ex.z, ex.w)));
                } else {
                  const float k4[4] = {kk.x, kk.y, kk.z, kk.w}, e4[4] = {ex.x, ex.y, ex.z, ex.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    t[j + e] = fmaf(capped(t[j + e] * k4[e], a.cap), kLog2e, e4[e]);
                }
                if (BIAS) {
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    t[j + e] = fmaf(-me.slope, fabsf(d - static_cast<float>(j + e)), t[j + e]);
                }
              }
              if (cut) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  t[j] = seen >> (h * 16 + j) & 1 ? t[j] : -INFINITY;
              }
#pragma unroll
              for (int j = 0; j < 16; j += 2)
                mx = fmax3(mx, t[j], t[j + 1]);
              tmem_st_32x16(t_s + c * 32 + h * 16, s[h]);
            }
          }
          tmem_st_wait();
          grown = mx > ref + kHeadroom;
          if (grown) {
            old = exp2f(ref - mx);
            ref = mx;
          }
          if (key0 > begin && __any_sync(0xffffffffu, grown)) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              tmem_ld_32x32(t_o + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j)
                o[j] = __float_as_uint(__uint_as_float(o[j]) * old);
              tmem_st_32x32(t_o + c * 32, o);
            }
            tmem_st_wait();
          }
          const float shift = kWeightLog2 - ref;
          const float2 shift2 = make_float2(shift, shift);
          float2 sum = make_float2(l * old, 0.f);
          tmem_ld_32x16(t_s, s[0]);
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t codes[16];      // e4m3 of 32 keys, then e5m2
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              tmem_ld_wait();
              if (h == 0 || c < 3)
                tmem_ld_32x16(t_s + c * 32 + (h + 1) * 16, s[h ^ 1]);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float4 inv = *reinterpret_cast<const float4*>(sc + 2 * kUnitKeys + c * 32 + h * 16 + 4 * j);
                const float* u = reinterpret_cast<const float*>(s[h]) + 4 * j;
                float2 x = fadd2(get2(u), shift2), y = fadd2(get2(u + 2), shift2);
                x = make_float2(exp2f(x.x), exp2f(x.y));
                y = make_float2(exp2f(y.x), exp2f(y.y));
                sum = ffma2(x, make_float2(inv.x, inv.y), sum);
                sum = ffma2(y, make_float2(inv.z, inv.w), sum);
                split_weights_e5m2(x, y, codes[h * 4 + j], codes[8 + h * 4 + j]);
              }
            }
            tmem_st_32x16(t_s + c * 32, codes);
          }
          tmem_st_wait();
          l = sum.x + sum.y;
        }
        if (key0 + kUnitKeys > end) {
          // rows of V behind the last key may hold any byte, a NaN times a weight of zero among them
          const int use = 2 * g + 1;
          mbar_wait(&full[use % kManyRing], (use / kManyRing) & 1, &abort_flag, p.status_word, 521);
          if (key0 + row >= end) {
            uint4* v = reinterpret_cast<uint4*>(ring + (use % kManyRing) * kTileBytes + row * kD);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              v[j] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        tc_fence_before_sync();
        fence_proxy_async_smem();
        warp_arrive(&p_full);
        warp_arrive(&sc_free[sl]);
      }
      warp_arrive(&q_free);      // all scores of the part have been taken
      // ---------------------------------------------------------------- the end of a part, 32 head dimensions at a time
      mbar_wait(&pv_done, (g - 1) & 1, &abort_flag, p.status_word, 522);
      tc_fence_after_sync();
      if (joined_parts > 1) {
        // the part goes to the workspace; fp8_join_kernel adds the parts of a tile up in their order
        float* mine = p.parts + static_cast<int64_t>(joined_slot) * kManyPart;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld_32x32(t_o + c * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j)      // a warp's rows lie side by side
            mine[(c * 32 + j) * kManyRows + row] = __uint_as_float(o[j]);
        }
        mine += kManyRows * kD + row;
        mine[0] = ref;
        mine[kManyRows] = l;
        if (joined_first) {
          mine[2 * kManyRows] = __int_as_float(me.out);
          mine[3 * kManyRows] = me.fix;
          if (tid == 0)
            p.joins[blockIdx.x] = joined_parts;
          owns = true;
        }
      } else if (alive) {
        const bool none = l == 0.f || me.fix == 0.f;
        const float mul = __fdividef(me.fix, l);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld_32x32(t_o + c * 32, o);
          tmem_ld_wait();
          // by way of shared memory: four lanes store the 64 bytes of a row
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              x[e] = none ? 0.f : __uint_as_float(o[8 * j + e]) * mul;
            *reinterpret_cast<uint4*>(out_stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = float_to_bf16x8(x);
          }
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = j * 8 + (lane >> 2);
            const int to = __shfl_sync(0xffffffffu, me.out, r);
            const uint4 v = *reinterpret_cast<const uint4*>(out_stage + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
            if (to >= 0)
              *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(to) * kD + c * 32 + (lane & 3) * 8) = v;
          }
          __syncwarp();
        }
      }
      tc_fence_before_sync();
      warp_arrive(&o_free);
    }
    if (tid == 0 && !owns)
      p.joins[blockIdx.x] = 0;
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kManyTmemCols);
  }
}

// Tiles whose parts lie in several CTAs of the many-rows kernel: the parts, in their order, added up.  A block has the tile that
// begins in CTA blockIdx.x (if one goes on from there) and eight head dimensions, a thread a row.  (The CTA that finishes last
// took 76 us to do this alone with 19 parts; blocks of 32 dimensions 15 us.)
constexpr int kJoinDims = 8;
__global__ void __launch_bounds__(kManyRows) fp8_join_kernel(const FewParams p) {
  pdl_wait();
  pdl_trigger();
  const int owner = blockIdx.x, row = threadIdx.x, c0 = blockIdx.y * kJoinDims;
  const int parts = __ldcg(p.joins + owner);
  if (parts == 0)
    return;
  const float* one = p.parts + (2 * static_cast<int64_t>(owner) + 1) * kManyPart + row;
  const float* rest = p.parts + 2 * static_cast<int64_t>(owner) * kManyPart + row;
  auto part = [&](int i) { return i == 0 ? one : rest + 2 * static_cast<int64_t>(i) * kManyPart; };
  constexpr int kRef = kManyRows * kD;
  const int out = __float_as_int(__ldcg(one + kRef + 2 * kManyRows));
  if (out < 0)
    return;
  float top = kNothing, l = 0.f, o[kJoinDims] = {};
#pragma unroll 4
  for (int i = 0; i < parts; ++i)
    top = fmaxf(top, __ldcg(part(i) + kRef));
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float* src = part(i);
    const float f = exp2f(__ldcg(src + kRef) - top);
    l = fmaf(__ldcg(src + kRef + kManyRows), f, l);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j] = fmaf(__ldcg(src + (c0 + j) * kManyRows), f, o[j]);
  }
  const float fix = __ldcg(one + kRef + 3 * kManyRows);
  const bool none = l == 0.f || fix == 0.f;
  const float mul = __fdividef(fix, l);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    o[j] = none ? 0.f : o[j] * mul;
  *reinterpret_cast<uint4*>(p.a.out + static_cast<int64_t>(out) * kD + c0) = float_to_bf16x8(o);
}

// Keys that any row of a tile sees; one warp per tile, numbered as Walk does.
template <int MROWS>
__global__ void __launch_bounds__(128) fp8_spans_kernel(const Fp8AttnParams p, int2* __restrict__ spans) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  const int lane = threadIdx.x & 31, group = p.H / p.Hkv;
  int number = blockIdx.x * 4 + (threadIdx.x >> 5);
  SeqWork w = {};
  for (int base = 0;; base += 32) {      // the tile's sequence
    if (base >= p.batch)
      return;
    const SeqWork x = seq_work<MROWS>(p, base + lane);
    const int upto = Walk<MROWS>::scan(x.tiles, lane);
    const unsigned hit = __ballot_sync(0xffffffffu, upto > number);
    if (hit) {
      const int src = __ffs(hit) - 1;
      number -= __shfl_sync(0xffffffffu, upto - x.tiles, src);
      w = seq_work<MROWS>(p, base + src);
      break;
    }
    number -= __shfl_sync(0xffffffffu, upto, 31);
  }
  int lo = w.len, hi = 0;
  const int t0 = number * MROWS, t1 = min(t0 + MROWS, w.rows);
  for (int i = t0 / group + lane; i <= (t1 - 1) / group; i += 32) {
    const int r = __ldg(p.idx + w.row0 + i);
    if (r < 0 || r >= p.total_q)
      continue;
    const int2 v = __ldg(p.ranges + r);
    const int x = max(v.x, 0), y = min(v.y, w.len);
    if (x < y) {
      lo = min(lo, x);
      hi = max(hi, y);
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  const int before = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (lane == 0)
    spans[before] = lo < hi ? make_int2(lo, hi) : make_int2(0, 0);
}

// Up to this many (listed row, query head) pairs a sequence and key head the few-rows kernel is the faster one, with a pass over
// the keys for each 32 of them: 26 rows (16 x 512 keys, 32 heads) 43 us against 63; 64 rows (8 x 4096 keys, 16 heads, capped) 125
// against 139; 128 rows (2 x 32011 keys, 8 key heads) 161 against 105.
constexpr int kFewMost = 64;

// Workspace: tickets, keys per tile (only with ranges), parts of tiles; for the kernel that needs most.
int64_t most_tiles(int num_salient, int batch, int group) { return static_cast<int64_t>(num_salient) * group / kRows + batch; }
size_t parts_offset(int64_t tiles, int ctas) { return (ctas * sizeof(unsigned long long) + tiles * sizeof(int2) + 255) / 256 * 256; }
size_t workspace_of(int num_salient, int batch, int group, int ctas) {
  const size_t few = 2ull * ctas * kRows * (kD + 2), many = 2ull * kManyCtas * ctas * kManyPart;
  return parts_offset(most_tiles(num_salient, batch, group), kManyCtas * ctas) +
         (static_cast<int64_t>(num_salient) * group > kFewMost ? max(few, many) : few) * sizeof(float);
}

template <typename Kernel>
int launch_rows(Kernel kernel, bool (&set)[64], int threads, uint32_t smem, const CUtensorMap& tk, const CUtensorMap& tv, const FewParams& p,
                int ctas, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  dev = (dev < 0 || dev >= 64) ? 0 : dev;
  if (!set[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
      return set_error(DYLLM_ERR_CUDA, "attention_salient_rows_fp8: cudaFuncSetAttribute failed: %s",
                       cudaGetErrorString(cudaGetLastError()));
    set[dev] = true;
  }
  DYLLM_LAUNCH(kernel, ctas, threads, smem, s, tk, tv, p);
  return check_launch("attention_salient_rows_fp8");
}
template <bool PLAIN>
int launch_few(const CUtensorMap& tk, const CUtensorMap& tv, const FewParams& p, int ctas, cudaStream_t s) {
  static bool set[64] = {};
  return launch_rows(fp8_few_rows_kernel<PLAIN>, set, kFewThreads, kFewSmem, tk, tv, p, ctas, s);
}
template <bool CAP, bool BIAS>
int launch_many(const CUtensorMap& tk, const CUtensorMap& tv, const FewParams& p, int ctas, cudaStream_t s) {
  static bool set[64] = {};
  const int rc = launch_rows(fp8_many_rows_kernel<CAP, BIAS>, set, kManyThreads, kManySmem, tk, tv, p, kManyCtas * ctas, s);
  if (rc != DYLLM_OK)
    return rc;
  DYLLM_LAUNCH(fp8_join_kernel, dim3(kManyCtas * ctas, kD / kJoinDims), kManyRows, 0, s, p);
  return check_launch("attention_salient_rows_fp8");
}

}  // namespace
}  // namespace dyllm

using namespace dyllm;

extern "C" {

size_t dyllm_attention_salient_rows_fp8_workspace_bytes(int num_salient, int batch, int num_heads, int num_kv_heads) {
  if (num_salient <= 0 || batch <= 0 || num_heads <= 0 || num_kv_heads <= 0)
    return 0;
  return workspace_of(num_salient, batch, num_heads / num_kv_heads, sm_count());
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
  DYLLM_REQUIRE(static_cast<int64_t>(num_salient) * num_heads < (1ll << 31), DYLLM_ERR_UNSUPPORTED,
                "attention_salient_rows_fp8: 2^31 output rows or more");
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
  const int ctas = sm_count();
  DYLLM_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, DYLLM_ERR_INVALID_ARGUMENT,
                "attention_salient_rows_fp8: the workspace must be 16-byte aligned");
  const int group = num_heads / num_kv_heads;
  const int64_t tiles = most_tiles(num_salient, batch, group);
  DYLLM_REQUIRE(workspace && workspace_bytes >= workspace_of(num_salient, batch, group, ctas), DYLLM_ERR_WORKSPACE,
                "attention_salient_rows_fp8: workspace of %zu bytes is smaller than the %zu required", workspace_bytes,
                workspace_of(num_salient, batch, group, ctas));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  f.a = p;
  f.tickets = reinterpret_cast<unsigned long long*>(ws);      // few rows
  f.joins = reinterpret_cast<int*>(ws);                       // many rows
  int2* spans = reinterpret_cast<int2*>(ws + kManyCtas * ctas * sizeof(unsigned long long));
  f.parts = reinterpret_cast<float*>(ws + parts_offset(tiles, kManyCtas * ctas));
  f.launch_id = next_launch_id() & ~0xffffull;
  f.status_word = device_status_word();
  // a sequence with more rows than the bound says is served by either kernel; so is one with few beside others with many
  const bool many = static_cast<int64_t>(max_rows_per_seq) * group > kFewMost && static_cast<int64_t>(num_salient) * group > kFewMost;
  if (p.ranges) {
    f.spans = spans;
    const unsigned blocks = static_cast<unsigned>((tiles + 3) / 4);
    if (many)
      DYLLM_LAUNCH(fp8_spans_kernel<kManyRows>, blocks, 128, 0, st, p, spans);
    else
      DYLLM_LAUNCH(fp8_spans_kernel<kRows>, blocks, 128, 0, st, p, spans);
  }
  CUtensorMap tk, tv;
  const uint64_t width = static_cast<uint64_t>(num_kv_heads) * kD;
  int rc = encode_tmap_2d_u8(&tk, k_codes, k_rows ? k_rows : 1, width, width, 32, kD);
  if (rc == DYLLM_OK)
    rc = encode_tmap_2d_u8(&tv, v_codes, v_rows ? v_rows : 1, width, width, 32, kD);
  if (rc != DYLLM_OK)
    return rc;
  if (many) {
    if (softcap > 0.f)
      return slopes ? launch_many<true, true>(tk, tv, f, ctas, st) : launch_many<true, false>(tk, tv, f, ctas, st);
    return slopes ? launch_many<false, true>(tk, tv, f, ctas, st) : launch_many<false, false>(tk, tv, f, ctas, st);
  }
  const bool plain = softcap == 0.f && !slopes && !key_ranges;
  return plain ? launch_few<true>(tk, tv, f, ctas, st) : launch_few<false>(tk, tv, f, ctas, st);
}

}  // extern "C"
