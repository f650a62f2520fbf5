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
  float scale, cap, inv_cap;   // cap in powers of two (times log2(e)), 1 / that
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

// Exponent of a value's scale (a power of two by definition).
__device__ __forceinline__ float value_exponent(float scale) {
  const uint32_t bits = __float_as_uint(scale);
  if (bits >= 0x7f800000u)
    return __uint_as_float(0x7fc00000u);
  return static_cast<float>(max(static_cast<int>(bits >> 23) - 127, kFp8MinExp));
}

constexpr int kUnitKeys = 128;                               // keys of a unit of work
constexpr int kRows = 32;                                    // rows of a tile of the few-rows kernel
constexpr int kParts = 4;                                    // slots of part descriptions
constexpr uint32_t kTileBytes = kUnitKeys * kD;
constexpr int kManyRows = 128;                               // and of the many-rows kernel
// A part in the workspace: [dimension][row] sums, [row] references, sums of weights; of a first part also output rows and `fix`.
__host__ __device__ constexpr int part_floats(int rows) { return rows * (kD + 4); }
constexpr int kFewPart = part_floats(kRows), kManyPart = part_floats(kManyRows);
constexpr float kWeightLog2 = 12.f;                          // the reference's weight: 2^12
constexpr float kHeadroom = 2.8f;                            // 2^(12 + 2.8) < 57344, the largest e5m2 number

struct WorkParams {
  Fp8AttnParams a;
  const int2* spans;           // per tile of rows: keys that any of them sees (null: all)
  unsigned long long* tickets; // one per CTA
  float* parts;                // two per CTA: [rows][128] sums, [rows] maxima, [rows] sums of weights
  int* joins;                  // per CTA: parts of the tile that begins in it and goes on in others (0: none); for fp8_join_kernel
  bool later;                  // that kernel joins them (of few rows: only where there are many parts)
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
// Walks over the parts of tiles that a CTA's share of the units consists of, in the order (sequence, tile, key head, keys).
// Uniform over a warp.
//
// Shares are cut at total * i / ctas, but no part of a tile is shorter than kMinPart units: a cut nearer to an end of its
// tile moves there, and a tile counts as kMinPart units at least (what it costs, too: most of a part's time passes before its second
// unit), so that no share is smaller: one sequence of 8192 keys among 70 of 100, 8 key heads, 46.7 us against 63.6 with 34 parts of one
// or two units; 32 x 601 ragged keys, 28 heads on 4, 28.6 against 35.0.  Joining the parts of a tile costs a CTA of the few-rows
// kernel about 5 us, a unit 3.  With many rows a unit takes 5 us and the join is a launch of its own: parts of at least 2 units
// against 4 take 34.6 us against 43.1 (32 x 601 keys, 28 heads on 4) and 163 against 166 (4 x 2048 rows of packed documents).
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
  static __device__ __forceinline__ int units_of(int2 span) { return max(kMinPart, (span.y - span.x + kUnitKeys - 1) / kUnitKeys); }
  // Units of a sequence's tiles, for one key head.
  static __device__ __forceinline__ int64_t seq_units(const WorkParams& p, const SeqWork& x, int base) {
    if (!p.spans)
      return static_cast<int64_t>(x.tiles) * units_of(make_int2(0, x.len));
    int64_t sum = 0;
    for (int t = 0; t < x.tiles; ++t)
      sum += units_of(__ldg(p.spans + base + t));
    return sum;
  }
  __device__ __forceinline__ void open(const WorkParams& p) {
    span = p.spans ? __ldg(p.spans + tile_base + tile) : make_int2(0, w.len);
    units = units_of(span);
  }
  __device__ __forceinline__ void start(const WorkParams& p) {
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
    ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total / kMinPart));
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
  __device__ __forceinline__ bool next(const WorkParams& p) {
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
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
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

// The same with B rows of 64 bytes (64-byte swizzle, groups of 8 rows 512 bytes apart).
__device__ __forceinline__ void umma_tile_b64(uint32_t d_tmem, uint32_t a_addr, uint32_t b_addr, uint32_t idesc, uint32_t accumulate) {
  constexpr uint32_t high = (1024u >> 4) | (1u << 14) | (2u << 29), high_b = (512u >> 4) | (1u << 14) | (4u << 29);
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\t"
      "mov.b64 b, {%2, %6};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"((a_addr >> 4) | (1u << 16)), "r"((b_addr >> 4) | (1u << 16)), "r"(idesc), "r"(accumulate), "n"(high), "n"(high_b)
      : "memory");
}

// A value that all lanes share, in a register of the uniform datapath: what depends on it alone (loop counters, descriptors)
// stays there, and an MMA issues every 33 cycles (its A operand's shared-memory read) instead of every 90.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }

// The team of 128 threads that works on a tile's rows (softmax of the few-rows kernel, loaders of the many-rows kernel) meets; any: whether the condition holds
// for one of them (after a wait that has given up they all leave together: a barrier would wait for those that are gone).
__device__ __forceinline__ void team_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool team_any(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x))
      : "memory");
  return r != 0;
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

constexpr float kNothing = -3.0e38f;      // maximum of no scores (finite: it takes part in differences; below every score)

// What a tile's rows are to the softmax warps.
struct RowInfo {
  int out;                     // output row, -1: none
  float fix;                   // 1; 0: the row does not exist in q; NaN: the query is not finite
  float mul;                   // scale of the query's codes (bits of its largest magnitude until that is worked out)
  float slope;                 // times log2(e)
  int pos, lo, hi;             // the row's place in its sequence, the keys that it sees
};

// The parts of a CTA's share one after the other, as the producer and the MMA warp walk over them.  Uniform over a warp.
struct PartWalk {
  int n, tiles;                // part, its units
  int begin, end, hk, k0, v0;
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
    tiles = (end - begin + kUnitKeys - 1) / kUnitKeys;
    return end >= 0;
  }
};

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
__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return floats2(r);
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return floats2(r);
}
// cap * tanh(s / cap).  With x = s / cap, below 1/4 (and for every score where the cap is large) the odd polynomial, of which
// 62/2835 x^8 < 2^-21 is left out; above, tanh(x) = 1 - 2 / (1 + e^2x), off by a few 2^-23, 2^-18 of a score at x = -1/4 and less
// further out.  (The hardware tanh has 2^-11; the second form alone is off by that much of the cap.)
__device__ __forceinline__ float2 capped(float2 s, float cap, float inv_cap) {
  const auto both = [](float v) { return make_float2(v, v); };
  const float2 x = fmul2(s, both(inv_cap)), u = fmul2(x, x), z = fmul2(x, both(2.f * kLog2e));
  float2 poly = ffma2(u, both(-17.f / 315.f), both(2.f / 15.f));
  poly = fmul2(ffma2(ffma2(poly, u, both(-1.f / 3.f)), u, both(1.f)), s);
  const float2 rest = make_float2(__fdividef(1.f, 1.f + exp2f(z.x)), __fdividef(1.f, 1.f + exp2f(z.y)));
  const float2 wide = ffma2(rest, both(-2.f * cap), both(cap));
  return make_float2(u.x < 0.0625f ? poly.x : wide.x, u.y < 0.0625f ? poly.y : wide.y);
}
// A row's reference for scores up to mx: weights are 2^(t - reference).  2^12 for the largest, but 1 where mx is so large (2^27) that
// their difference would be rounded up past the largest e5m2 number.
__device__ __forceinline__ float reference(float mx) {
  const float ref = mx - kWeightLog2;
  return mx - ref > kHeadroom + kWeightLog2 ? mx : ref;
}
// The lowest n bits.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// Four weights, rounded to half precision (2^-11), as three codes in e5m2 each, which are the high bytes of half-precision numbers:
// the number, what that leaves, what that leaves, the first two rounded by adding half a step.  Eleven bits in three codes of three
// bits and two signs: their sum is the half-precision number, exactly down to 2^-6 (below, the last one's steps of 2^-16).
__device__ __forceinline__ void split_weights(float2 a, float2 b, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const __half2 x[2] = {__floats2half2_rn(a.x, a.y), __floats2half2_rn(b.x, b.y)};
  uint32_t h[2], m[2], l[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    h[i] = *reinterpret_cast<const uint32_t*>(&x[i]) + 0x00800080u;
    const uint32_t u = h[i] & 0xff00ff00u;
    const __half2 r = __hsub2(x[i], *reinterpret_cast<const __half2*>(&u));
    m[i] = *reinterpret_cast<const uint32_t*>(&r) + 0x00800080u;
    const uint32_t v = m[i] & 0xff00ff00u;
    const __half2 q = __hsub2(r, *reinterpret_cast<const __half2*>(&v));      // a NaN ends up here
    l[i] = *reinterpret_cast<const uint32_t*>(&q);
  }
  hi = __byte_perm(h[0], h[1], 0x7531);
  mid = __byte_perm(m[0], m[1], 0x7531);
  lo = __byte_perm(l[0], l[1], 0x7531);
}

// ----------------------------------------------------------------------------------------------
// Few rows per sequence: bound by the bytes of the cache, which go from the TMA ring to the tensor cores as they are, and by the
// chain of steps from the lists of a sequence to its result.
//
// The rows of a tile are up to 32 (listed row, query head) pairs of one sequence and key head, so that grouped query heads share
// one pass over their keys.  A unit of work is 128 keys of a tile; all units of the launch, in the order (sequence, tile, key head,
// keys), are dealt out to the CTAs in equal contiguous shares that every CTA works out for itself from the device-side counts.  A
// tile whose units lie in several CTAs is joined by the CTA that finishes last, or where there will be many parts by a launch of
// its own, in the order of its parts.
//
// The products are transposed, keys (then head dimensions) in the M = 128 of tcgen05.mma.kind::f8f6f4:
//   S^T = K Q^T         A: K tile as loaded (K-major), B: the queries as e4m3 + e5m2, two products into one accumulator
//   O^T = V^T P^T       A: V tile as loaded (MN-major), B: the weights as three codes in e5m2, three products into one accumulator
// A query in bf16 (8 significant bits) is e4m3 (4 bits) plus a remainder of at most 3 bits in e5m2, next to a power of two of its own
// row: exact down to 2^-14.8 of the row's largest element (below that e4m3 runs out of bits), off by 2^-21.8 of it at most.  A
// weight is 2^12 * 2^(t - reference) in half precision, as with many rows: off by 2^-11 of itself or by 2^-28 of the largest.  (As
// e4m3 + e5m2 it was off by 2^-8 of itself, or by 2^-20 of the largest: percents of what many small weights beside a large one make
// up together; 32.0 us for 34.4 at the size below.  Codes cut instead of rounded, 2^-8.4 of a weight: 32.8; conversion instructions
// instead of added half steps: 34.8.)  The codes of the cache are never widened.
//
// Four softmax warps, thread = key with the scores of all rows in registers; a row's reference is in shared memory and follows the
// maximum in steps, so that a unit costs one barrier (does any score exceed its reference by more than 2.8?) and the maxima are
// looked for only where one does.  A part of four units takes 14 us from its description to its result, nearly all of it waits
// along that chain, so four CTAs per SM with parts of their own take turns: 16 x 512 keys, 32 heads, 26 rows take 33 us (2.3 TB/s
// of the cache).  With the weights of before 30 us, and then 41 us with three CTAs, where 68 of 512 tiles wait for a second turn, 43 us
// with one CTA of sixteen softmax warps.
// ----------------------------------------------------------------------------------------------
constexpr int kFewRing = 2;                                  // slots of one K or V tile
constexpr int kFewCtas = 4;                                  // per SM
constexpr int kFewWarps = 4, kFewThreads = 32 * (3 + kFewWarps);
constexpr uint32_t kFewTmemCols = 128, kQBytes = kRows * kD, kPBytes = kUnitKeys * 64;
constexpr uint32_t kP3Bytes = kPBytes / 2;
constexpr uint32_t kFewSmem = kFewRing * kTileBytes + kPBytes + 2 * kQBytes + kP3Bytes + 1024;      // four CTAs per SM have 55 KB each with the static part

// Sum of each of 32 values over the lanes of a warp: lane l gets that of value l.
__device__ __forceinline__ float sum_lanes(float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int half = 16; half; half >>= 1) {
    const bool upper = lane & half;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float give = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, half);
    }
  }
  return v[0];
}

// CAP, BIAS: scores capped by a tanh, biased by their distance.
template <bool CAP, bool BIAS>
__global__ void __launch_bounds__(kFewThreads, kFewCtas)
fp8_few_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const WorkParams p) {
  pdl_wait();      // programmatic dependent launch: nothing before this reads an earlier kernel's data
  pdl_trigger();
  const Fp8AttnParams& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* p_smem = ring + kFewRing * kTileBytes;            // first and second codes of the weights: [128 keys][32, 32], 64-byte swizzle
  uint8_t* q_smem = p_smem + kPBytes;                        // [32 rows][128] e4m3, then e5m2
  uint8_t* p3_smem = q_smem + 2 * kQBytes;                   // third codes of the weights: [64][keys 0 .., keys 64 .. of 32], 64-byte swizzle
  __shared__ uint64_t full[kFewRing], empty[kFewRing], part_full[kParts], part_done[kParts], q_asked, q_full, s_full[2], p_full, pv_done, o_free;
  __shared__ PartInfo s_part[kParts];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, joins;
  __shared__ int s_out[kRows];                               // output row, -1: none
  __shared__ int2 s_sees[kRows], s_all[kFewWarps];           // keys that a row sees, that all rows see (of a quarter of them)
  __shared__ __align__(16) float2 s_bias[kRows];             // slope times log2(e), place in the sequence counted from the part's first key
  __shared__ __align__(16) float s_fix[kRows], s_mul[kRows], s_max[kFewWarps][kRows], s_ref[kFewWarps][kRows], s_old[kFewWarps][kRows];      // a copy for each warp
  float (&s_sum)[kFewWarps][kRows] = s_max;                  // the maxima have been read once a part's last unit has been multiplied
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kFewRing; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kParts; ++i) {
      mbar_init(&part_full[i], 1);
      mbar_init(&part_done[i], kFewWarps + 2);
    }
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(&p_full, kFewWarps);
    mbar_init(&pv_done, 1);
    mbar_init(&q_asked, kFewWarps);
    mbar_init(&q_full, kFewWarps);
    mbar_init(&o_free, kFewWarps);
    fence_mbar_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kFewTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;      // S^T of two units, 32 columns each, then O^T

  if (warp == 2) {
    // ---------------------------------------------------------------- scheduler: the parts of this CTA's share
    Walk<kRows> walk;
    walk.start(p);
    for (int n = 0;;) {
      const bool more = walk.next(p);
      const int slot = n % kParts;
      if (n >= kParts && !mbar_wait(&part_done[slot], (n / kParts - 1) & 1, &abort_flag, p.status_word, 400))
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
    // ---------------------------------------------------------------- producer: K of a unit before V of the last
    int n = 0;
    bool asked = false;
    PartWalk c = {};
    auto load = [&](const CUtensorMap* map, int row0, int key) {
      const int slot = n % kFewRing;
      if (n >= kFewRing)
        mbar_wait(&empty[slot], (n / kFewRing - 1) & 1, &abort_flag, p.status_word, 401);
      if (elect_one()) {
        const int boxes = min(4, (c.end - key + 31) / 32);      // no box of keys that do not belong to the part
        mbar_arrive_expect_tx(&full[slot], boxes * 32 * kD);
        for (int j = 0; j < boxes; ++j)
          tma_load_2d(ring + slot * kTileBytes + j * 32 * kD, map, &full[slot], c.hk * kD, row0 + key + 32 * j);
      }
      __syncwarp();
      ++n;
    };
    for (bool more = c.open(part_full, part_done, s_part, &abort_flag, p.status_word); more;) {
      if (c.tiles && !asked) {
        // the first part's rows before the tiles, which would hold them up (8 x 4096 keys, 64 rows 93.0 -> 90.8 us)
        asked = true;
        mbar_wait(&q_asked, 0, &abort_flag, p.status_word, 403);
      }
      if (c.tiles)
        load(&tmap_k, c.k0, c.begin);
      for (int key = c.begin; key < c.end; key += kUnitKeys) {
        if (key + kUnitKeys < c.end)
          load(&tmap_k, c.k0, key + kUnitKeys);
        load(&tmap_v, c.v0, key);
      }
      ++c.n;
      more = c.open(part_full, part_done, s_part, &abort_flag, p.status_word);
    }
    // a CTA may not end with copies on their way, also when a wait of another warp has given up
    for (int i = max(0, n - kFewRing); i < n; ++i)
      mbar_wait(&full[i % kFewRing], (i / kFewRing) & 1, &abort_flag, p.status_word, 402);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer: scores of a unit before the sums of the last
    constexpr uint32_t idesc_hi = umma_idesc_f8(128, kRows, 0, 0, 0, 0), idesc_lo = umma_idesc_f8(128, kRows, 0, 1, 0, 0);
    constexpr uint32_t idesc_pv = umma_idesc_f8(128, kRows, 0, 1, 1, 1);
    const uint32_t ring_addr = smem_u32(ring), p_addr = smem_u32(p_smem), q_addr = smem_u32(q_smem), p3_addr = smem_u32(p3_smem), t_s = uniform(tmem), t_o = t_s + 64;
    int n = 0, u0 = 0, live = 0;      // tiles of the ring, units before the part, parts that have some
    PartWalk c = {};
    auto scores = [&](int i) {
      const int slot = n % kFewRing, u = u0 + i;
      mbar_wait(&full[slot], (n / kFewRing) & 1, &abort_flag, p.status_word, 405);
      tc_fence_after_sync();
      if (elect_one()) {
        const uint32_t k_addr = ring_addr + slot * kTileBytes, d = t_s + (u & 1) * kRows;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {      // 32 head dimensions = 32 bytes a step
          umma_tile(d, k_addr + 32 * kk, q_addr + 32 * kk, idesc_hi, kk != 0 ? 1u : 0u);
          umma_tile(d, k_addr + 32 * kk, q_addr + kQBytes + 32 * kk, idesc_lo, 1u);
        }
        umma_commit(&empty[slot]);
        umma_commit(&s_full[u & 1]);
      }
      __syncwarp();
      ++n;
    };
    for (bool more = c.open(part_full, part_done, s_part, &abort_flag, p.status_word); more;) {
      if (c.tiles) {
        mbar_wait(&q_full, live & 1, &abort_flag, p.status_word, 403);
        scores(0);
      }
      for (int i = 0; i < c.tiles; ++i) {
        if (i + 1 < c.tiles)
          scores(i + 1);      // into the columns whose scores became the weights that the last product took
        const int slot = n % kFewRing, u = u0 + i;
        mbar_wait(&full[slot], (n / kFewRing) & 1, &abort_flag, p.status_word, 406);
        if (i == 0 && live > 0)
          mbar_wait(&o_free, (live - 1) & 1, &abort_flag, p.status_word, 408);
        mbar_wait(&p_full, u & 1, &abort_flag, p.status_word, 407);
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t v_addr = ring_addr + slot * kTileBytes;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {      // 32 keys: 32 rows of V and of the weights
            umma_tile_b64(t_o, v_addr + kk * 4096, p_addr + kk * 2048, idesc_pv, (i | kk) != 0 ? 1u : 0u);
            umma_tile_b64(t_o, v_addr + kk * 4096, p_addr + 32 + kk * 2048, idesc_pv, 1u);
            umma_tile_b64(t_o, v_addr + kk * 4096, p3_addr + 32 * (kk >> 1) + (kk & 1) * 2048, idesc_pv, 1u);
          }
          umma_commit(&empty[slot]);
          umma_commit(&pv_done);
        }
        __syncwarp();
        ++n;
      }
      live += c.tiles ? 1 : 0;
      u0 += c.tiles;
      ++c.n;
      more = c.open(part_full, part_done, s_part, &abort_flag, p.status_word);
    }
  } else {
    // ---------------------------------------------------------------- softmax over the keys, epilogue
    const int quarter = warp & 3;                  // tensor-memory lanes: keys (head dimensions) 32 * quarter ..
    const int tid = threadIdx.x - 96;
    const int kl = quarter * 32 + lane;            // key of a unit, or head dimension
    const int group = a.H / a.Hkv;
    const uint32_t t_s = tmem + (static_cast<uint32_t>(quarter * 32) << 16), t_o = t_s + 64;
    int u = 0, n_ring = 0;                         // units and tiles of the ring so far
    if (p.later && tid == 0)
      p.joins[blockIdx.x] = 0;                     // unless a tile begins here that goes on in other CTAs
    for (int n = 0;; ++n) {
      if (team_any(!mbar_wait(&part_full[n % kParts], (n / kParts) & 1, &abort_flag, p.status_word, 415)))
        break;
      const PartInfo part = s_part[n % kParts];
      warp_arrive(&part_done[n % kParts]);
      const int begin = part.begin, end = part.end;
      if (end < 0)
        break;
      if (end == begin) {      // no keys: zeros
        for (int t = part.t0 + (tid >> 4); t < min(part.t0 + kRows, part.rows); t += 8) {
          const int i = t / group;
          const int64_t row = (static_cast<int64_t>(part.row0) + i) * a.H + part.hk * group + t - i * group;
          *reinterpret_cast<uint4*>(a.out + row * kD + (tid & 15) * 8) = make_uint4(0u, 0u, 0u, 0u);
        }
        continue;
      }
      const float* k_scale = a.k_scales + static_cast<int64_t>(part.k0) * a.Hkv + part.hk;
      const float* v_scale = a.v_scales + static_cast<int64_t>(part.v0) * a.Hkv + part.hk;
      float ks_next = 1.f, vs_next = 1.f;
      if (begin + kl < end) {
        ks_next = __ldg(k_scale + static_cast<int64_t>(begin + kl) * a.Hkv);
        vs_next = __ldg(v_scale + static_cast<int64_t>(begin + kl) * a.Hkv);
      }
      // queries: eight threads a row, rows tid / 8 and 16 + tid / 8; codes next to the row's own largest element, e4m3 and the e5m2
      // rest
      {
        uint4 x0[2], x1[2];
        int at[2], head[2], t[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          t[h] = part.t0 + 16 * h + (tid >> 3);
          const int i = t[h] / group;
          head[h] = part.hk * group + t[h] - i * group;
          at[h] = t[h] < part.rows ? __ldg(a.idx + part.row0 + i) : -1;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          at[h] = at[h] >= a.total_q ? -1 : at[h];
          x0[h] = x1[h] = make_uint4(0u, 0u, 0u, 0u);
          if (at[h] >= 0) {
            const uint4* src = reinterpret_cast<const uint4*>(a.q + at[h] * a.ldq + head[h] * kD) + (tid & 7) * 2;
            x0[h] = __ldg(src);
            x1[h] = __ldg(src + 1);
          }
        }
        if (u == 0)
          warp_arrive(&q_asked);
        int2 sees = make_int2(0, end);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 16 * h + (tid >> 3);
          uint32_t top = fp8_amax8(max(bf16x8_amax(x0[h]), bf16x8_amax(x1[h])));
          const bool finite = top < 0x7f800000u;
          if (!finite) {
            x0[h] = x1[h] = make_uint4(0u, 0u, 0u, 0u);
            top = 0;
          }
          const uint32_t scale = fp8_scale_bits(top);
          uint4 hi, lo;
          split_query(x0[h], x1[h], fp8_inverse(scale), hi, lo);
          uint8_t* dst = q_smem + r * kD + (((tid & 7) ^ (r & 7)) << 4);
          *reinterpret_cast<uint4*>(dst) = hi;
          *reinterpret_cast<uint4*>(dst + kQBytes) = lo;
          if ((tid & 7) == 0) {
            s_out[r] = t[h] < part.rows ? (part.row0 + t[h] / group) * a.H + head[h] : -1;
            // 1; 0: the row does not exist in q; NaN: the query is not finite
            s_fix[r] = at[h] < 0 ? 0.f : finite ? 1.f : __uint_as_float(0x7fc00000u);
            s_mul[r] = __uint_as_float(scale);
            if (BIAS && at[h] >= 0) {
              const int pos = __ldg(a.cu_k + part.b + 1) - __ldg(a.cu_k + part.b) - (__ldg(a.cu_q + part.b + 1) - at[h]);
              s_bias[r] = make_float2(__ldg(a.slopes + head[h]) * kLog2e, static_cast<float>(pos - begin));
            } else {
              s_bias[r] = make_float2(0.f, 0.f);
            }
            if (a.ranges && at[h] >= 0) {
              const int2 range = __ldg(a.ranges + at[h]);
              s_sees[r] = make_int2(max(range.x, 0), min(range.y, end));
              sees.x = max(sees.x, range.x);
              sees.y = min(sees.y, range.y);
            } else {
              s_sees[r] = make_int2(0, end);
            }
          }
        }
        sees.x = __reduce_max_sync(0xffffffffu, sees.x);
        sees.y = __reduce_min_sync(0xffffffffu, sees.y);
        if (lane == 0)
          s_all[quarter] = sees;
        fence_proxy_async_smem();
        warp_arrive(&q_full);
        team_sync();
      }
      const float key_mul = a.scale * kLog2e;      // scores and caps are taken times log2(e)
      const int all_from = max(max(s_all[0].x, s_all[1].x), max(s_all[2].x, s_all[3].x));
      const int all_to = min(min(s_all[0].y, s_all[1].y), min(s_all[2].y, s_all[3].y));
      const int tiles = (end - begin + kUnitKeys - 1) / kUnitKeys;
      float l = 0.f;                               // lane = row: sum of the weights of this quarter's keys
      float was = kNothing;                        // lane = row: reference, as in s_ref
      float* my_ref = s_ref[quarter];
      for (int i = 0; i < tiles; ++i, ++u) {
        const int at = begin + i * kUnitKeys + kl, buf = u & 1;
        const float kk = ks_next * key_mul, ex = value_exponent(vs_next), place = static_cast<float>(at - begin);
        if (at + kUnitKeys < end) {
          ks_next = __ldg(k_scale + static_cast<int64_t>(at + kUnitKeys) * a.Hkv);
          vs_next = __ldg(v_scale + static_cast<int64_t>(at + kUnitKeys) * a.Hkv);
        }
        mbar_wait(&s_full[buf], (u >> 1) & 1, &abort_flag, p.status_word, 409);
        tc_fence_after_sync();
        uint32_t s[kRows];
        float* t = reinterpret_cast<float*>(s);
        tmem_ld_32x32(t_s + buf * kRows, s);
        tmem_ld_wait();
        // scores (times log2 e, plus the exponents of the values' scales)
#pragma unroll
        for (int r = 0; r < kRows; r += 4) {
          // the factors of row and key first: their product is within the type's range wherever the score is
          const float4 row = *reinterpret_cast<const float4*>(s_mul + r);
          const float2 m0 = fmul2(make_float2(row.x, row.y), make_float2(kk, kk)), m1 = fmul2(make_float2(row.z, row.w), make_float2(kk, kk));
          if (CAP) {
            put2(t + r, fadd2(capped(fmul2(get2(t + r), m0), a.cap, a.inv_cap), make_float2(ex, ex)));
            put2(t + r + 2, fadd2(capped(fmul2(get2(t + r + 2), m1), a.cap, a.inv_cap), make_float2(ex, ex)));
          } else {
            put2(t + r, ffma2(get2(t + r), m0, make_float2(ex, ex)));
            put2(t + r + 2, ffma2(get2(t + r + 2), m1, make_float2(ex, ex)));
          }
          if (BIAS) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float4 b = *reinterpret_cast<const float4*>(s_bias + r + e);
              t[r + e] = fmaf(-b.x, fabsf(b.y - place), t[r + e]);
              t[r + e + 1] = fmaf(-b.z, fabsf(b.w - place), t[r + e + 1]);
            }
          }
        }
        if (at - kl < all_from || at - kl + kUnitKeys > all_to) {      // not all rows see all keys
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const int2 sees = s_sees[r];
            t[r] = at >= sees.x && at < sees.y ? t[r] : -INFINITY;
          }
        }
        // does any lie above its reference by more than the weights' codes can take?
        bool moves = i == 0;
        if (!moves) {
          float above = -INFINITY;
#pragma unroll
          for (int r = 0; r < kRows; r += 4) {
            const float4 ref = *reinterpret_cast<const float4*>(my_ref + r);
            above = fmax3(above, t[r] - ref.x, t[r + 1] - ref.y);
            above = fmax3(above, t[r + 2] - ref.z, t[r + 3] - ref.w);
          }
          moves = team_any(above > kHeadroom + kWeightLog2);
        }
        if (moves) {
          float mx = 0.f;
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const float m = warp_max(t[r]);
            mx = lane == r ? m : mx;
          }
          s_max[quarter][lane] = mx;
          team_sync();
          mx = fmaxf(fmaxf(s_max[0][lane], s_max[1][lane]), fmaxf(s_max[2][lane], s_max[3][lane]));
          const float ref = mx - was > kHeadroom + kWeightLog2 ? reference(mx) : was, old = exp2f(was - ref);
          l *= old;
          was = ref;
          my_ref[lane] = ref;
          s_old[quarter][lane] = old;
          __syncwarp();
          if (i > 0) {
            mbar_wait(&pv_done, (u - 1) & 1, &abort_flag, p.status_word, 410);
            tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < kRows; c += 8) {
              uint32_t o[8];
              tmem_ld_32x8(t_o + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int r = 0; r < 8; ++r)
                o[r] = __float_as_uint(__uint_as_float(o[r]) * s_old[quarter][c + r]);
              tmem_st_32x8(t_o + c, o);
            }
            tmem_st_wait();
          }
        }
        // weights
        if (u > 0)
          mbar_wait(&pv_done, (u - 1) & 1, &abort_flag, p.status_word, 411);      // the last ones have been taken
        uint8_t* dst = p_smem + kl * 64;
        uint8_t* dst3 = p3_smem + (kl & 63) * 64;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t hi[4], mid[4], lo[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 16 * h + 4 * j;
            const float4 ref = *reinterpret_cast<const float4*>(my_ref + r);
            t[r] = exp2f(t[r] - ref.x);
            t[r + 1] = exp2f(t[r + 1] - ref.y);
            t[r + 2] = exp2f(t[r + 2] - ref.z);
            t[r + 3] = exp2f(t[r + 3] - ref.w);
            split_weights(make_float2(t[r], t[r + 1]), make_float2(t[r + 2], t[r + 3]), hi[j], mid[j], lo[j]);
          }
          *reinterpret_cast<uint4*>(dst + ((h ^ (kl >> 1 & 3)) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(dst + (((2 + h) ^ (kl >> 1 & 3)) << 4)) = make_uint4(mid[0], mid[1], mid[2], mid[3]);
          *reinterpret_cast<uint4*>(dst3 + (((2 * (kl >> 6) + h) ^ (kl >> 1 & 3)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        if (at - kl + kUnitKeys > end) {
          // rows of V behind the last key may hold any byte, a NaN times a weight of zero among them
          const int use = n_ring + 2 * i + 1;      // the part's last tile in the ring
          mbar_wait(&full[use % kFewRing], (use / kFewRing) & 1, &abort_flag, p.status_word, 412);
          if (at >= end) {
            uint4* v = reinterpret_cast<uint4*>(ring + (use % kFewRing) * kTileBytes + kl * kD);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              v[j] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        tc_fence_before_sync();
        fence_proxy_async_smem();
        warp_arrive(&p_full);
        // the weight of a NaN is a NaN where its key is seen, else zero
        const float inv = ex == ex ? exp2f(-ex) : 1.f;
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          t[r] *= inv;
        float (&w)[kRows] = *reinterpret_cast<float (*)[kRows]>(s);
        l += sum_lanes(w);
      }
      n_ring += 2 * tiles;

      // ---------------------------------------------------------------- thread = head dimension kl of all rows
      const float fix = s_fix[lane];
      float top = was;
      mbar_wait(&pv_done, (u - 1) & 1, &abort_flag, p.status_word, 413);
      tc_fence_after_sync();
      s_sum[quarter][lane] = l;
      uint32_t ou[kRows];
      float* o = reinterpret_cast<float*>(ou);
      tmem_ld_32x32(t_o, ou);
      tmem_ld_wait();
      tc_fence_before_sync();
      warp_arrive(&o_free);
      team_sync();
      l = (s_sum[0][lane] + s_sum[1][lane]) + (s_sum[2][lane] + s_sum[3][lane]);
      bool store = true;
      if (part.parts > 1) {
        float* mine = p.parts + static_cast<int64_t>(part.slot) * kFewPart;
#pragma unroll
        for (int r = 0; r < kRows; r += 4)
          *reinterpret_cast<float4*>(mine + kl * kRows + r) = make_float4(o[r], o[r + 1], o[r + 2], o[r + 3]);
        if (quarter == 0) {
          mine[kRows * kD + lane] = top;
          mine[kRows * kD + kRows + lane] = l;
        }
        if (p.later) {
          store = false;
          if (part.first && quarter == 0) {
            mine[kRows * kD + 2 * kRows + lane] = __int_as_float(s_out[lane]);
            mine[kRows * kD + 3 * kRows + lane] = fix;
          }
          if (part.first && tid == 0)
            p.joins[blockIdx.x] = part.parts;
        } else {
          __threadfence();
          team_sync();
          if (tid == 0) {
            open_join(p.tickets + part.owner, p.launch_id);
            joins = last_to_join(p.tickets + part.owner, part.parts) ? 1 : 0;
          }
          team_sync();
          store = joins != 0;
        }
        if (store) {
          __threadfence();
          const float* first = p.parts + (2 * static_cast<int64_t>(part.owner) + 1) * kFewPart;
          const float* rest = p.parts + 2 * static_cast<int64_t>(part.owner) * kFewPart;
          top = kNothing;
          l = 0.f;
#pragma unroll
          for (int r = 0; r < kRows; ++r)
            o[r] = 0.f;
          for (int i = 0; i < part.parts; ++i)
            top = fmaxf(top, __ldcg((i == 0 ? first : rest + 2 * static_cast<int64_t>(i) * kFewPart) + kRows * kD + lane));
          for (int i = 0; i < part.parts; ++i) {
            const float* src = i == 0 ? first : rest + 2 * static_cast<int64_t>(i) * kFewPart;
            const float f = exp2f(__ldcg(src + kRows * kD + lane) - top);
            l = fmaf(__ldcg(src + kRows * kD + kRows + lane), f, l);
#pragma unroll
            for (int r = 0; r < kRows; r += 4) {
              const float4 v = __ldcg(reinterpret_cast<const float4*>(src + kl * kRows + r));
              o[r] = fmaf(v.x, __shfl_sync(0xffffffffu, f, r), o[r]);
              o[r + 1] = fmaf(v.y, __shfl_sync(0xffffffffu, f, r + 1), o[r + 1]);
              o[r + 2] = fmaf(v.z, __shfl_sync(0xffffffffu, f, r + 2), o[r + 2]);
              o[r + 3] = fmaf(v.w, __shfl_sync(0xffffffffu, f, r + 3), o[r + 3]);
            }
          }
        }
      }
      if (store) {
        // by way of shared memory, where weights and queries were: 16 threads store the 256 bytes of a row
        float* lines = reinterpret_cast<float*>(p_smem);
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          lines[r * kD + kl] = o[r];
        if (quarter == 0)
          s_old[0][lane] = l == 0.f || fix == 0.f ? 0.f : __fdividef(fix, l);
        team_sync();
#pragma unroll
        for (int r = tid >> 4; r < kRows; r += 8) {
          const int out = s_out[r];
          const float mul = s_old[0][r];
          if (out >= 0) {
            float x[8];
            *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(lines + r * kD + (tid & 15) * 8);
            *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(lines + r * kD + (tid & 15) * 8 + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              x[e] = mul == 0.f ? 0.f : x[e] * mul;
            *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(out) * kD + (tid & 15) * 8) = float_to_bf16x8(x);
          }
        }
      }
      team_sync();      // nobody overwrites the rows or what describes them while another warp reads it
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kFewTmemCols);
  }
}

// ----------------------------------------------------------------------------------------------
// Many rows per sequence: bound by the passes over tensor memory and the instructions around the exponentials.  A unit of 128 rows x
// 128 keys takes the tensor cores 1250 cycles, its exponentials 1024, the scales of its keys (three words a key for each of four
// warps) 1536 of shared memory; with all else it takes an SM 5100 (2 x 32011 keys, 128 pairs a key head: 112 us, of which 9 for lists
// and queries, 5 for the join).  Without the reads of the scales it would take 89 us, without the scores' pass 86, without the
// weights' pass 86, without the products of the third codes 110.
//
// Tiles of 128 (listed row, query head) pairs, rows in the M = 128 of the products:
//   S = Q K^T    A: the queries as e4m3 + e5m2 (two products into one accumulator), B: the K tile as loaded (K-major)
//   O = P V      A: the weights as three codes in e5m2, B: the V tile as loaded (MN-major)
// Thread = row in four softmax warps.  A weight is 2^12 * 2^(t - reference); the reference follows the maximum in steps, so that the
// sums are rescaled only where a score lies more than 2.8 (log2) above it.  A weight is off by 2^-11 of itself or by 2^-28 of the
// largest.  Scores and weights share 128 columns of tensor memory (the three codes of 32 keys' weights lie in the first 24 of their
// scores' 32 columns), so the steps of one tile follow one another; two CTAs per SM, each with parts of its own, fill each other's
// waits, the ends of parts among them.  Four loader warps stage the queries of the next part and the scales of the next tiles.
// ----------------------------------------------------------------------------------------------
constexpr int kManyRing = 4;                                 // slots of one K or V tile
constexpr int kScaleSlots = 2;                               // tiles whose scales are staged ahead
constexpr int kManyWarps = 4, kManyThreads = 32 * (3 + kManyWarps + 4);
constexpr int kManyCtas = 2;                                 // per SM
// (Dynamic, static and the system's shared memory of two CTAs leave 128 bytes: more of it, and there is one CTA per SM, 157 us for 110.)
constexpr uint32_t kManyTmemCols = 256;
constexpr uint32_t kStageBytes = 32 * 64;                    // of a softmax warp: 32 head dimensions of its rows
constexpr uint32_t kManyQBytes = kManyRows * kD;             // e4m3 or e5m2 part of the queries of a tile
constexpr uint32_t kManySmem = kManyRing * kTileBytes + 2 * kManyQBytes + kManyWarps * kStageBytes +
                               kScaleSlots * 3 * kUnitKeys * sizeof(float) + 1024;


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
fp8_many_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const WorkParams p) {
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
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ RowInfo s_row[kManyRows];
  __shared__ int64_t s_src[kManyRows];
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
    PartWalk c = {};
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
    constexpr uint32_t idesc_pv = umma_idesc_f8(128, 128, 1, 0, 0, 1);
    const uint32_t ring_addr = smem_u32(ring), q_addr = smem_u32(q_smem), t_s = uniform(tmem), t_o = t_s + 128;
    int g = 0, live = 0;      // tiles, parts that have some
    PartWalk c = {};
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
          for (int kk = 0; kk < 4; ++kk) {      // 32 keys: three times 8 columns of weights, 32 rows of V
            umma_tile_ts(t_o, t_s + 32 * kk, v_addr + kk * 4096, idesc_pv, i == 0 && kk == 0 ? 0u : 1u);
            umma_tile_ts(t_o, t_s + 32 * kk + 8, v_addr + kk * 4096, idesc_pv, 1u);
            umma_tile_ts(t_o, t_s + 32 * kk + 16, v_addr + kk * 4096, idesc_pv, 1u);
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
      const int slot = n % kParts;
      if (team_any(!mbar_wait(&part_full[slot], (n / kParts) & 1, &abort_flag, p.status_word, 510)))
        break;
      const PartInfo w = s_part[slot];
      team_sync();
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
            const int2 range = __ldg(a.ranges + at);      // cut: differences with keys must not wrap
            v.lo = max(range.x, 0);
            v.hi = max(min(range.y, w.len), 0);
          }
        }
      }
      if (w.end == w.begin) {      // no keys: zeros
        s_src[tid] = v.out;
        team_sync();
#pragma unroll 1
        for (int r = tid >> 4; r < kManyRows; r += 8)
          if (s_src[r] >= 0)
            *reinterpret_cast<uint4*>(a.out + s_src[r] * kD + (tid & 15) * 8) = make_uint4(0u, 0u, 0u, 0u);
        team_sync();
        continue;
      }
      // the first tile's scales are on their way with the queries
      const float* ks = a.k_scales + static_cast<int64_t>(w.k0) * a.Hkv + w.hk;
      const float* vs = a.v_scales + static_cast<int64_t>(w.v0) * a.Hkv + w.hk;
      float first_k = 1.f, first_v = 1.f;
      if (w.begin + tid < w.end) {
        first_k = __ldg(ks + static_cast<int64_t>(w.begin + tid) * a.Hkv);
        first_v = __ldg(vs + static_cast<int64_t>(w.begin + tid) * a.Hkv);
      }
      s_src[tid] = src;
      team_sync();
      // queries: eight threads a row, 16 rows at a time, four times 16 in flight; codes next to the row's own largest element.
      // (Loops: straight-line code for 128 rows that runs once a part costs more in instruction fetches than it saves.)
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
      const float mul = a.scale * kLog2e;      // scores (but for the row's factor) and caps are taken times log2(e)
      auto deposit = [&](float k, float v) {
        const int sl = n_sc % kScaleSlots;
        if (n_sc >= kScaleSlots)
          mbar_wait(&sc_free[sl], (n_sc / kScaleSlots - 1) & 1, &abort_flag, p.status_word, 512);
        const float ex = value_exponent(v);
        float* dst = sc_smem + sl * 3 * kUnitKeys + tid;
        dst[0] = k * mul;
        dst[kUnitKeys] = ex;
        dst[2 * kUnitKeys] = ex == ex ? exp2f(-ex) : 1.f;      // the weight of a NaN is a NaN where its key is seen, else zero
        warp_arrive(&sc_full[sl]);
        ++n_sc;
      };
      fetch(0);
      deposit(first_k, first_v);
      if (live > 0)
        mbar_wait(&q_free, (live - 1) & 1, &abort_flag, p.status_word, 511);
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        if (h)
          fetch(h);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 64 * h + 16 * k + (tid >> 3), part = tid & 7;
          const uint32_t top = fp8_amax8(max(bf16x8_amax(x0[k]), bf16x8_amax(x1[k])));
          if (part == 0)
            s_row[r].mul = __uint_as_float(top);
          if (top >= 0x7f800000u)
            x0[k] = x1[k] = make_uint4(0u, 0u, 0u, 0u);
          uint4 hi, lo;
          split_query(x0[k], x1[k], fp8_inverse(fp8_scale_bits(top)), hi, lo);
          uint8_t* dst = q_smem + r * kD + ((part ^ (r & 7)) << 4);
          *reinterpret_cast<uint4*>(dst) = hi;
          *reinterpret_cast<uint4*>(dst + kManyQBytes) = lo;
        }
      }
      team_sync();
      const uint32_t top = __float_as_uint(s_row[tid].mul);
      if (top >= 0x7f800000u)
        v.fix = __uint_as_float(0x7fc00000u);
      v.mul = __uint_as_float(fp8_scale_bits(top >= 0x7f800000u ? 0u : top));
      s_row[tid] = v;
      fence_proxy_async_smem();
      team_sync();
      warp_arrive(&q_full);
      ++live;
      // scales of the other tiles: thread = key, four tiles' loads at a time
      for (int key = w.begin + kUnitKeys + tid; key - tid < w.end; key += 4 * kUnitKeys) {
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
          if (key - tid + i * kUnitKeys < w.end)
            deposit(x[i], y[i]);
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
    if (tid == 0)
      p.joins[blockIdx.x] = 0;        // unless a tile begins here that goes on in other CTAs
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
                // the factors of row and key first: their product is within the type's range wherever the score is
                const float2 f = fmul2(make_float2(kk.x, kk.y), make_float2(me.mul, me.mul)), g2 = fmul2(make_float2(kk.z, kk.w), make_float2(me.mul, me.mul));
                if (!CAP) {
                  put2(t + j, ffma2(get2(t + j), f, make_float2(ex.x, ex.y)));
                  put2(t + j + 2, ffma2(get2(t + j + 2), g2, make_float2(ex.z, ex.w)));
                } else {
                  put2(t + j, fadd2(capped(fmul2(get2(t + j), f), a.cap, a.inv_cap), make_float2(ex.x, ex.y)));
                  put2(t + j + 2, fadd2(capped(fmul2(get2(t + j + 2), g2), a.cap, a.inv_cap), make_float2(ex.z, ex.w)));
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
          grown = mx - ref > kHeadroom + kWeightLog2;
          if (grown) {
            old = ref;
            ref = reference(mx);
            old = exp2f(old - ref);
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
          const float2 shift2 = make_float2(-ref, -ref);
          float2 sum = make_float2(l * old, 0.f);
          tmem_ld_32x16(t_s, s[0]);
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t codes[16], third[8];      // first codes of 32 keys, second, third
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
                split_weights(x, y, codes[h * 4 + j], codes[8 + h * 4 + j], third[h * 4 + j]);
              }
            }
            tmem_st_32x16(t_s + c * 32, codes);
            tmem_st_32x8(t_s + c * 32 + 16, third);
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
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kManyTmemCols);
  }
}

// Tiles whose parts lie in several CTAs: the parts, in their order, added up.  A block has the tile that begins in CTA blockIdx.x
// (if one goes on from there), a thread a row and eight head dimensions.  (The CTA that finishes last took 76 us to do this alone
// with 19 parts of 128 rows; blocks of 32 dimensions 15 us.)
constexpr int kJoinThreads = 128, kJoinDims = 8;
template <int ROWS>
__global__ void __launch_bounds__(kJoinThreads) fp8_join_kernel(const WorkParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int kPart = part_floats(ROWS);
  const int owner = blockIdx.x, row = threadIdx.x % ROWS, c0 = (blockIdx.y * (kJoinThreads / ROWS) + threadIdx.x / ROWS) * kJoinDims;
  const int parts = __ldcg(p.joins + owner);
  if (parts == 0)
    return;
  const float* one = p.parts + (2 * static_cast<int64_t>(owner) + 1) * kPart + row;
  const float* rest = p.parts + 2 * static_cast<int64_t>(owner) * kPart + row;
  auto part = [&](int i) { return i == 0 ? one : rest + 2 * static_cast<int64_t>(i) * kPart; };
  constexpr int kRef = ROWS * kD;
  const int out = __float_as_int(__ldcg(one + kRef + 2 * ROWS));
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
    l = fmaf(__ldcg(src + kRef + ROWS), f, l);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j] = fmaf(__ldcg(src + (c0 + j) * ROWS), f, o[j]);
  }
  const float fix = __ldcg(one + kRef + 3 * ROWS);
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

// The kernel for a call.  Up to kFewMost (listed row, query head) pairs a sequence and key head the few-rows kernel is taken, with a
// pass over the keys for each 32 of them; so it is for more of them where the caches are short (their rows are all that the host
// knows of the keys): tiles of up to 8 units, which it does not split, and at most ten units a CTA.  Few against many, us:
//   26 pairs (16 x 512 keys, 32 heads) 33 : 66; 64 there 57 : 72; 64 over 8 x 4096 keys 97 : 109, capped 111 : 150; over 2 x 32011 92 : 103
//   77 (175 keys, 4 key heads) 13 : 21; 84 (32 x 601, 4) 27 : 36; 140 there 43 : 46; 96 (2 x 1001, 8) 25 : 26
//   96 (2 x 32011 keys, 8 key heads) 119 : 105, biased 133 : 110; 90 (16 x 512, 32) 82 : 74; 128 there 106 : 77
constexpr int kFewMost = 64;
bool takes_many(int64_t max_rows, int64_t num_salient, int64_t batch, int64_t group, int64_t kv_heads, int64_t cache_rows, int64_t ctas) {
  const int64_t most = min(max_rows, num_salient) * group;
  if (most <= kFewMost)
    return false;
  const int64_t tiles = (min(most, (num_salient * group + batch - 1) / batch) + kRows - 1) / kRows;
  return cache_rows > 8 * kUnitKeys * batch || (cache_rows / kUnitKeys + batch) * tiles * kv_heads > 10 * kFewCtas * ctas;
}

// Whether the few-rows kernel leaves the joins to a launch: where a tile of average length will have more than six parts.  The CTA
// that finishes last adds them up in 1 us each: 2 x 32011 keys, 8 key heads, 32 pairs (37 parts) 121 us against 72 with the launch,
// 64 pairs (18 parts) 112 against 84.
bool joins_later(int64_t max_rows, int64_t num_salient, int64_t batch, int64_t group, int64_t kv_heads, int64_t cache_rows, int64_t ctas) {
  const int64_t most = min(min(max_rows, num_salient) * group, (num_salient * group + batch - 1) / batch);
  const int64_t tiles = (most + kRows - 1) / kRows * batch * kv_heads;
  return min(cache_rows / kUnitKeys / batch / kMinPartFew, kFewCtas * ctas / tiles) > 6;
}

// The kernels of a call: the few-rows or the many-rows one, that of the spans, that of the joins.
struct Kernels {
  bool many, spans, join;
  int count() const { return 1 + spans + join; }
};
Kernels kernels_of(int num_salient, int batch, int max_rows, int heads, int kv_heads, int64_t cache_rows, bool ranges, int ctas) {
  // a sequence with more rows than the bound says is served by either kernel; so is one with few beside others with many
  const bool many = takes_many(max_rows, num_salient, batch, heads / kv_heads, kv_heads, cache_rows, ctas);
  return {many, ranges, many || joins_later(max_rows, num_salient, batch, heads / kv_heads, kv_heads, cache_rows, ctas)};
}

// Workspace: tickets, keys per tile (only with ranges), parts of tiles; for the kernel that needs most.
constexpr int kMostCtas = kFewCtas > kManyCtas ? kFewCtas : kManyCtas;
int64_t most_tiles(int num_salient, int batch, int group) { return static_cast<int64_t>(num_salient) * group / kRows + batch; }
size_t parts_offset(int64_t tiles, int ctas) { return (ctas * sizeof(unsigned long long) + tiles * sizeof(int2) + 255) / 256 * 256; }
size_t workspace_of(int num_salient, int batch, int group, int ctas) {
  const size_t few = 2ull * kFewCtas * ctas * kFewPart, many = 2ull * kManyCtas * ctas * kManyPart;
  return parts_offset(most_tiles(num_salient, batch, group), kMostCtas * ctas) +
         (static_cast<int64_t>(num_salient) * group > kFewMost ? max(few, many) : few) * sizeof(float);
}

// CTAs of a launch: no more than there can be parts, whatever the counts on the device say (one request of 256 keys: 32 CTAs
// instead of 592, 11.0 us instead of 11.7).
int grid_of(const Fp8AttnParams& a, int tile_rows, int min_part, int most) {
  const int64_t tiles = (static_cast<int64_t>(a.num_salient) * (a.H / a.Hkv) / tile_rows + a.batch) * a.Hkv;
  const int64_t parts = max(tiles, tiles * (a.k_rows / kUnitKeys + 1) / min_part);
  return static_cast<int>(min(static_cast<int64_t>(most), parts));
}

template <typename Kernel>
int launch_rows(Kernel kernel, bool (&set)[64], int threads, uint32_t smem, const CUtensorMap& tk, const CUtensorMap& tv, const WorkParams& p,
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
template <int ROWS>
int launch_join(const WorkParams& p, int ctas, cudaStream_t s) {
  DYLLM_LAUNCH(fp8_join_kernel<ROWS>, dim3(ctas, kD / kJoinDims * ROWS / kJoinThreads), kJoinThreads, 0, s, p);
  return check_launch("attention_salient_rows_fp8");
}
template <bool CAP, bool BIAS>
int launch_few(const CUtensorMap& tk, const CUtensorMap& tv, const WorkParams& p, int ctas, cudaStream_t s) {
  static bool set[64] = {};
  const int grid = grid_of(p.a, kRows, kMinPartFew, kFewCtas * ctas);
  const int rc = launch_rows(fp8_few_rows_kernel<CAP, BIAS>, set, kFewThreads, kFewSmem, tk, tv, p, grid, s);
  return rc == DYLLM_OK && p.later ? launch_join<kRows>(p, grid, s) : rc;
}
template <bool CAP, bool BIAS>
int launch_many(const CUtensorMap& tk, const CUtensorMap& tv, const WorkParams& p, int ctas, cudaStream_t s) {
  static bool set[64] = {};
  const int grid = grid_of(p.a, kManyRows, kMinPartMany, kManyCtas * ctas);
  const int rc = launch_rows(fp8_many_rows_kernel<CAP, BIAS>, set, kManyThreads, kManySmem, tk, tv, p, grid, s);
  return rc == DYLLM_OK ? launch_join<kManyRows>(p, grid, s) : rc;
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

int dyllm_attention_salient_rows_fp8_launches(int num_salient, int batch, int max_rows_per_seq, int num_heads, int num_kv_heads,
                                              int64_t k_rows, int has_key_ranges) {
  if (num_salient <= 0 || batch <= 0 || max_rows_per_seq <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return 0;
  return kernels_of(num_salient, batch, max_rows_per_seq, num_heads, num_kv_heads, k_rows, has_key_ranges != 0, sm_count()).count();
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
  // a smaller cap: its quotient may be infinite, and a score of zero times that is no number; a larger one: its quotient is not normal
  DYLLM_REQUIRE(scale == scale && (softcap == 0.f || softcap >= 1e-6f) && softcap <= 0x1p125f, DYLLM_ERR_INVALID_ARGUMENT,
                "attention_salient_rows_fp8: scale %g softcap %g", static_cast<double>(scale), static_cast<double>(softcap));
  if (batch == 0 || num_salient == 0 || max_rows_per_seq == 0)
    return DYLLM_OK;
  // empty tensors have no address, and nothing reads them
  DYLLM_REQUIRE((q || total_q == 0) && ((k_codes && k_scales) || k_rows == 0) && ((v_codes && v_scales) || v_rows == 0) && k_seq_starts &&
                    v_seq_starts && seq_ids && out && cu_seqlens_q && cu_seqlens_k && cu_salientlens && idx_salient_row,
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
  p.cap = softcap * kLog2e;
  p.inv_cap = softcap > 0.f ? 1.f / p.cap : 0.f;
  p.slopes = slopes;
  p.ranges = reinterpret_cast<const int2*>(key_ranges);
  WorkParams f = {};
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
  f.tickets = reinterpret_cast<unsigned long long*>(ws);
  f.joins = reinterpret_cast<int*>(ws);                       // or these
  int2* spans = reinterpret_cast<int2*>(ws + kMostCtas * ctas * sizeof(unsigned long long));
  f.parts = reinterpret_cast<float*>(ws + parts_offset(tiles, kMostCtas * ctas));
  f.launch_id = next_launch_id() & ~0xffffull;
  f.status_word = device_status_word();
  const Kernels kernels = kernels_of(num_salient, batch, max_rows_per_seq, num_heads, num_kv_heads, k_rows, p.ranges != nullptr, ctas);
  const bool many = kernels.many;
  f.later = kernels.join;
  if (kernels.spans) {
    f.spans = spans;
    const unsigned blocks = static_cast<unsigned>((tiles + 3) / 4);
    if (many)
      DYLLM_LAUNCH(fp8_spans_kernel<kManyRows>, blocks, 128, 0, st, p, spans);
    else
      DYLLM_LAUNCH(fp8_spans_kernel<kRows>, blocks, 128, 0, st, p, spans);
  }
  CUtensorMap tk, tv;
  const uint64_t width = static_cast<uint64_t>(num_kv_heads) * kD;
  // (a cache without rows: a descriptor that no copy uses)
  int rc = encode_tmap_2d_u8(&tk, k_rows ? k_codes : out, k_rows ? k_rows : 1, width, width, 32, kD);
  if (rc == DYLLM_OK)
    rc = encode_tmap_2d_u8(&tv, v_rows ? v_codes : out, v_rows ? v_rows : 1, width, width, 32, kD);
  if (rc != DYLLM_OK)
    return rc;
  if (softcap > 0.f) {
    if (slopes)
      return many ? launch_many<true, true>(tk, tv, f, ctas, st) : launch_few<true, true>(tk, tv, f, ctas, st);
    return many ? launch_many<true, false>(tk, tv, f, ctas, st) : launch_few<true, false>(tk, tv, f, ctas, st);
  }
  if (slopes)
    return many ? launch_many<false, true>(tk, tv, f, ctas, st) : launch_few<false, true>(tk, tv, f, ctas, st);
  return many ? launch_many<false, false>(tk, tv, f, ctas, st) : launch_few<false, false>(tk, tv, f, ctas, st);
}

}  // extern "C"
