// sample_requests.cu — a token for each request of a step, with its own temperature, top-k, top-p,
// min-p and random number (gq_sample_requests).
//
//   w_i = e^((l_i - max l) / T)
//   in the order of the logits (largest first, ties to the smaller id): the first top_k; of those the
//   shortest run that holds top_p of their mass; of those the ones with w_i >= min_p
//   token: in the order of the ids, the first kept one at which the running sum of w passes u * (their sum)
//
// All three options keep a beginning of the order, so what is left is one border: a logit and an id,
// together a key of 64 bits. It is found without sorting: a histogram of counts (top-k) or masses (top-p) over
// 2048 bins (4096 of a whole row's first) says in which bin the border lies, and that bin is cut again until few keys
// are left to be compared. Nor are all of a row's keys needed, mostly: three launches.
//   survey  a CTA per piece of a row, for all SMs to read the logits: its largest, its largest keys (as many as
//           make some 1024 of a row), and its sum of masses where the whole row's counts
//   finish  a CTA per row, among the keys that the pieces have given; without top-k, top-p and min-p there are
//           no keys: the piece in which the sum passes u of the whole, and the token in it
//   last    a cluster of CTAs per row, for the rows whose border is below what the pieces have given (a top_p
//           of a flat distribution, more equal logits than there is room for) or whose largest is infinite
// Masses are whole numbers, w * 2^44 rounded: their sums (vocab <= 2^19) fit 64 bits and do not depend on
// the order of additions, so atomics may add them up. The weights are made in f64: with f32's 2^-24 a
// draw over 262144 tokens would land on a neighbour of the right token every few hundred rows; 2^-45
// leaves less than one in 10^6.
//
// 64 rows of 262144 logits, 67 MB, 10 us of memory traffic: 29 us with a top_k of 64, 32 with a top_p of
// 0.95 of those or a top_k of 1000, 55 over all tokens, 85 of mixed options (survey 28, finish 20, last 37 for
// three of the rows); one row 13 to 19 us, 45 where its border lies far down. The survey has its issue slots 68%
// taken (53% of the time with its ends, f64 18%), and its pieces take turns; the finish is dependent steps of one CTA a
// row (up to three searches in turn, issue 41%), and so is the last launch: passes over a CTA's columns with six cluster
// barriers between, 33 us a row (issue 22%; code that is not at the SM yet, barriers and loads are waited for most).
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "gq_internal.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;     // of the second and the last launch
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;  // (of the last launch's CTAs: see there)
constexpr int kBins = 2048;
constexpr int kFirst = 2 * kBins; // of a row's first round: sums of 32 bits
constexpr int kOne = 44;          // w = 1 is 2^44
constexpr int kLimb = 15;         // bits of a mass that one 32-bit sum takes: a CTA has at most 2^15 columns
constexpr int kMaxShare = 32768;  // columns of a CTA
constexpr int kList = 2048;       // keys of a row that the last launch lists
constexpr int kFew = 256;         // keys that are compared with one another
constexpr int kGiven = 1024;      // keys that a row's pieces give together, about; a larger top_k has twice as many
constexpr int kMostGiven = 4096;  // and no more
constexpr int kSurvey = 256;      // threads that survey a piece
constexpr int kMaxPiece = 8192;   // (a thread's 32 columns: a bit each; with 4096 as the most, mixed options take 90 us in place of 85)
static_assert(kMaxPiece <= 32 * kSurvey);
constexpr int kRows = 256;        // rows of a launch
constexpr int kTable = 16;
static_assert(kMaxShare <= 64 * kThreads);  // (a thread's columns: a bit each)
constexpr int64_t kMaxVocab = (int64_t)kMaxShare * kMaxCluster;
constexpr int kMaxPieces = 128;

// 2^(j / 16)
__constant__ double kPowers[kTable] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
    1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
    1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
    1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

struct Args {
  const float *logits;
  int64_t ld;
  int vocab, share;  // share: columns of a CTA
  int run;           // columns of a warp, a multiple of 128; kWarps * run >= share
  int wide;          // rows are read 16 bytes at a time
  const float *temperature, *top_p, *min_p;
  const int32_t *top_k;
  const double *uniforms;
  uint64_t *rng;
  int32_t *tokens;
  float *probs;
  // what the first launch finds in each piece of a row
  int pieces, piece, give;  // of a row; columns of a piece; the most keys of one
  float *piece_top, *piece_from;
  uint64_t *piece_mass, *piece_keys;
  int32_t *piece_given, *todo, *n_todo;  // todo: rows that are left to the last launch; how many, and how many it has begun
  double *drawn;       // the row's random number
  uint64_t *row_mass;  // all of a row's, where top_p asks for it
  uint32_t *err;
};

// What a CTA works with by itself.
struct Scratch {
  union {
    uint32_t limb[3][kBins];  // sums of a mass's bits 0-14, 15-29 and 30-44 (counts: the first)
    uint64_t bin[kBins];      // the same as one number
    uint32_t first[kFirst];   // two to a word of those
    uint64_t list[kList];     // keys of some bins
    struct {
      uint64_t few[kFew], few_mass[kFew];
    };
  };
  double table[kTable];  // 2^(j / 16): 128 bytes, a lane's entry is on banks of its own
  uint64_t warp_sum[kWarps];
  uint64_t border, border_mass, total, need, range[2][kWarps];
  uint32_t bin_at, bin_to, count;
};

// With what the CTAs of a cluster exchange.
struct Shared : Scratch {
  uint64_t whole[kBins];  // the bins of the whole row, then the keys of all CTAs' lists: written by every CTA
  uint64_t masses[kList]; // of those keys
  uint64_t part[kThreads];
  uint64_t cta_sum[kMaxCluster];  // written by every CTA, as is this:
  uint32_t cta_count[kMaxCluster];
  int turn;
  unsigned long long kept[kWarps];  // masses of the warps' columns that are kept
  float warp_top[kWarps], warp_from[kWarps];
};
static_assert(kBins >= kList && kBins >= 2 * kMaxCluster);

// Order of the logits as an order of numbers (no logit is NaN here, and no zero negative).
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}
// Of a logit and its id: larger logits first, then smaller ids.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t id) { return ((uint64_t)key_of(v) << 32) | (uint32_t)~id; }

// A row's largest logit (a number here), and what a weight is made with.
struct Row {
  float top, least;  // from `least` down a mass is 0
  bool far;          // `least` is -inf: -inf has to be told apart
  double scale;      // 16 log2(e) / T
};
__device__ __forceinline__ Row row_of(float top, float t) {  // t > 0, or 0 for the limit
  Row row;
  row.top = top;
  // the largest number that is 32 T and more below: e^-32 * 2^44 is below 1/2
  row.least = top - 33.0f * t;
  if ((double)top - (double)row.least < 32.0 * (double)t || t == 0.0f) row.least = nextafterf(row.least, -INFINITY);
  row.far = row.least == -INFINITY;
  const double gap = (double)top - (double)row.least;
  row.scale = kTable * 1.4426950408889634074 / (double)t;
  // (where a rounding of `top` is much more than T, nothing lies between the two)
  if (!row.far && gap > 128.0 * (double)t) row.scale = 48.0 * kTable / gap;
  if (row.far && t == 0.0f) row.scale = 0.0;
  return row;
}

// 2^52 plus w * 2^44 to the nearest whole number: 2^(t / 16), t = j + r with |r| <= 1/2, is 2^(j / 16) from a
// table times a Taylor polynomial of degree 6 (its next term is below 2^-50). The last addition rounds.
constexpr double kWhole = 4503599627370496.0;
__device__ __forceinline__ double rounded_mass(const double *table, const Row &row, float v) {
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
  constexpr double c = 0.69314718055994530942 / kTable;
  const double x = (double)fmaxf(v, row.least) - (double)row.top;
  const double whole = fma(x, row.scale, kRound);
  const int j = __double2loint(whole);
  const double r = fma(x, row.scale, kRound - whole);
  double p = fma(r, c * c * c * c * c * c / 720, c * c * c * c * c / 120);
  p = fma(r, p, c * c * c * c / 24);
  p = fma(r, p, c * c * c / 6);
  p = fma(r, p, c * c / 2);
  p = fma(r, p, c);
  p = fma(r, p, 1.0);
  p *= table[j & (kTable - 1)];
  p = __hiloint2double(__double2hiint(p) + ((j >> 4) + kOne) * (1 << 20), __double2loint(p));
  return p + kWhole;
}
__device__ __forceinline__ uint64_t mass_of(const double *table, const Row &row, float v) {
  const double m = rounded_mass(table, row, v);
  const uint64_t w = ((uint64_t)(__double2hiint(m) & 0xfffff) << 32) | (uint32_t)__double2loint(m);
  return row.far && v == -INFINITY ? 0 : w;
}

// (called, where a key's mass is made by itself: code that runs once is bound by being fetched)
__device__ __noinline__ uint64_t mass_of_key(const double *table, const Row row, uint64_t key) { return mass_of(table, row, logit_of(key)); }
__device__ __forceinline__ uint64_t bits_of(double m) { return (uint64_t)__double_as_longlong(m); }
constexpr uint64_t kWholeBits = 0x4330000000000000ull;  // of kWhole: the bits of kWhole + m are these plus m

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t warp_scan(uint64_t v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t up = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += up;
  }
  return v;
}
// Inclusive scan over the block; sums[] of scratch. The total too.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *sums, uint64_t &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan(v);
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) v += sums[i];
    total += sums[i];
  }
  __syncthreads();
  return v;
}

// Of two logits and ids: whether the first is at or ahead of the second in the order.
__device__ __forceinline__ bool from_on(float v, uint32_t id, float v0, uint32_t id0) { return v > v0 || (v == v0 && id <= id0); }

// A NaN is never drawn: -inf. -0 counts as 0.
__device__ __forceinline__ float4 clean(float4 v) {
  return make_float4(fmaxf(v.x, -INFINITY) + 0.0f, fmaxf(v.y, -INFINITY) + 0.0f, fmaxf(v.z, -INFINITY) + 0.0f, fmaxf(v.w, -INFINITY) + 0.0f);
}
// Four logits of a row from column c on, -inf past its n columns, as they are.
__device__ __forceinline__ float4 raw_logits(const float *row, int c, int n, bool wide) {
  float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  if (wide && c + 3 < n) {
    v = *reinterpret_cast<const float4 *>(row + c);
  } else {
    if (c < n) v.x = row[c];
    if (c + 1 < n) v.y = row[c + 1];
    if (c + 2 < n) v.z = row[c + 2];
    if (c + 3 < n) v.w = row[c + 3];
  }
  return v;
}

// A lane's columns of a row: four from `id` on, four 128 on, ... (n times). The passes over them are functions
// of their own, so that each has the registers that it needs.
struct Columns {
  const float *row;
  int n, end, share;  // end: of this CTA's columns, share of them
  uint32_t id;
  bool wide, infinite;  // infinite: the row's largest is +inf; such logits become 0, the others -inf
  __device__ __forceinline__ float4 at(int i) const {
    float4 v = clean(raw_logits(row, (int)id + i * 128, end, wide));
    if (infinite)
      v = make_float4(v.x == INFINITY ? 0.0f : -INFINITY, v.y == INFINITY ? 0.0f : -INFINITY, v.z == INFINITY ? 0.0f : -INFINITY,
                      v.w == INFINITY ? 0.0f : -INFINITY);
    return v;
  }
};

// A lane's columns one after another, the next two on their way.
struct Stream {
  const Columns &c;
  float4 ahead[2];
  __device__ __forceinline__ explicit Stream(const Columns &columns) : c(columns) {
    ahead[0] = c.at(0);
    ahead[1] = c.at(1);
  }
  __device__ __forceinline__ float4 take(int i) {  // i = 0, 1, ..., c.n - 1 (what is read past those is not used)
    const float4 x = ahead[0];
    ahead[0] = ahead[1];
    ahead[1] = c.at(i + 2);
    return x;
  }
};

// Where the border may be, and the bin of a logit there. (Ends are keys and compared as such: a bin's end need not be
// a logit's key, and there is one among them that stands for -0, which as a logit were equal to 0.)
struct Span {
  uint64_t low, high;   // the last and the first key
  int shift;            // -1: bins by the distance from the largest logit; else by (high - key) >> shift
  float top, per_logit;
  // (rounded by the addition; only the order matters, and that equal logits have equal bins)
  __device__ __forceinline__ uint32_t first_bin(float v) const {
    return __float_as_uint(fminf((top - v) * per_logit, (float)(kFirst - 1)) + 8388608.0f) & (kFirst - 1);
  }
  __device__ __forceinline__ bool has(float v, uint32_t id) const {
    const uint64_t key = rank_key(v, id);
    return v > -INFINITY && key >= low && key <= high;
  }
  __device__ __forceinline__ uint32_t key_bin(float v, uint32_t id) const { return (uint32_t)((high - rank_key(v, id)) >> shift); }
};

// Adds to shared memory what is not 0 (a predicate, no branch).
__device__ __forceinline__ void add_some(uint32_t *to, uint32_t v) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p red.shared.add.u32 [%0], %1;\n\t}" ::"r"(gqd::smem_u32(to)), "r"(v) : "memory");
}
__device__ __forceinline__ void add_mass(uint32_t (*limb)[kBins], uint32_t b, uint64_t w) {
  const uint32_t rest = (uint32_t)(w >> kLimb);
  add_some(&limb[0][b], (uint32_t)w & ((1u << kLimb) - 1));
  add_some(&limb[1][b], rest & ((1u << kLimb) - 1));
  add_some(&limb[2][b], rest >> kLimb);
}

// The first round's bins: all numbers (counts), or those from a border on (masses).
__device__ __noinline__ void count_bins(const Columns c, const Span p, uint32_t *count) {
  Stream next(c);
#pragma unroll 2
  for (int i = 0; i < c.n; ++i) {
    const float4 x = next.take(i);
    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      add_some(&count[p.first_bin(v[k])], v[k] > -INFINITY);
  }
}
// Masses to some 2^-17, as shares of 2^31 of the whole: which bins the border can be in.
template <bool LOW>
__device__ __noinline__ void share_bins(const Columns c, const Span p, float rate, float unit, uint32_t *sum) {
  const float low_v = logit_of(p.low);
  const uint32_t low_id = ~(uint32_t)p.low;
  Stream next(c);
#pragma unroll 1
  for (int i = 0; i < c.n; ++i) {
    const float4 x = next.take(i);
    const float v[4] = {x.x, x.y, x.z, x.w};
    const uint32_t id = c.id + i * 128;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float w;  // (halves: a difference of two numbers may be infinite)
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"((0.5f * v[k] - 0.5f * p.top) * rate));
      if (v[k] == p.top) w = 1.0f;
      const bool in = v[k] > -INFINITY && (!LOW || from_on(v[k], id + k, low_v, low_id));
      add_some(&sum[p.first_bin(v[k])], in ? __float2uint_rn(w * unit) : 0u);
    }
  }
}
// A later round's.
template <bool MASS>
__device__ __noinline__ void key_bins(const Columns c, const Span p, const Row row, const double *table, uint32_t (*limb)[kBins]) {
  Stream next(c);
#pragma unroll 1
  for (int i = 0; i < c.n; ++i) {
    const float4 x = next.take(i);
    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
      const uint32_t id = c.id + i * 128 + k;
      const float l = k == 0 ? v[0] : k == 1 ? v[1] : k == 2 ? v[2] : v[3];
      if (!p.has(l, id)) continue;
      if (MASS) add_mass(limb, p.key_bin(l, id), mass_of(table, row, l));
      else atomicAdd(&limb[0][p.key_bin(l, id)], 1u);
    }
  }
}
// The keys of some bins to this CTA's list (kList at most). The masses of the bins ahead of those (SUM) are
// added up. (LOW: the span has an end.)
template <bool FIRST, bool SUM, bool LOW>
__device__ __noinline__ uint64_t collect(const Columns c, const Span p, const Row row, const double *table, uint32_t bin, uint32_t last,
                                         uint64_t *list, uint32_t *listed) {
  const int lane = threadIdx.x & 31;
  uint64_t sum = 0, mark = 0;  // a bit for each of the lane's columns
  const float low_v = logit_of(p.low);  // (FIRST and LOW: a logit's key)
  const uint32_t low_id = ~(uint32_t)p.low;
  Stream next(c);
#pragma unroll 1
  for (int i = 0; i < c.n; ++i) {
    const float4 x = next.take(i);
    const float v[4] = {x.x, x.y, x.z, x.w};
    const uint32_t id = c.id + i * 128;
    uint32_t in = 0, ahead = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (FIRST) {
        const uint32_t b = p.first_bin(v[k]);
        const bool from = v[k] > -INFINITY && (!LOW || from_on(v[k], id + k, low_v, low_id));
        in |= (uint32_t)(b >= bin && b <= last && from) << k;
        if (SUM) ahead |= (uint32_t)(b < bin && v[k] > row.least && from) << k;
      } else {
        in |= (uint32_t)(p.has(v[k], id + k) && p.key_bin(v[k], id + k) == bin) << k;
      }
    }
    mark |= (uint64_t)in << (4 * i);
    if (SUM && __any_sync(0xffffffffu, ahead)) {
      double m[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) m[k] = rounded_mass(table, row, v[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += ahead >> k & 1 ? bits_of(m[k]) - kWholeBits : 0;
    }
  }
  const uint32_t own = __popcll(mark);
  uint32_t to = own, from = 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, to, o);
    if (lane >= o) to += up;
  }
  if (lane == 31 && to > 0) from = atomicAdd(listed, to);
  to += __shfl_sync(0xffffffffu, from, 31) - own;
  for (; mark && to < (uint32_t)kList; mark &= mark - 1, ++to) {
    const int at = __ffsll((long long)mark) - 1;
    const uint32_t id = c.id + (at >> 2) * 128 + (at & 3);
    list[to] = rank_key(c.infinite ? 0.0f : c.row[id] + 0.0f, id);
  }
  return sum;
}

// One number for each of this CTA's bins.
template <bool MASS>
__device__ __forceinline__ void join_limbs(Scratch &s) {
  uint64_t w[kBins / kThreads];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBins / kThreads; ++i) {
    const int b = threadIdx.x + i * kThreads;
    w[i] = MASS ? s.limb[0][b] + ((uint64_t)s.limb[1][b] << kLimb) + ((uint64_t)s.limb[2][b] << (2 * kLimb)) : s.limb[0][b];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBins / kThreads; ++i) s.bin[threadIdx.x + i * kThreads] = w[i];
}

// The bin in which the sum of bins, from the first on, reaches what is needed, and what is needed of it; and the
// bin in which it reaches more (`to`). PAIRS: of the first round's.
template <bool PAIRS>
__device__ __forceinline__ void find_bin(Scratch &s, const uint64_t *bins, uint64_t &need, uint64_t to, uint32_t &bin, uint32_t &last) {
  constexpr int kEach = (PAIRS ? kFirst : kBins) / kThreads;
  uint64_t w[kEach], mine = 0, total;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    mine += w[i] = PAIRS ? reinterpret_cast<const uint32_t *>(bins)[threadIdx.x * kEach + i] : bins[threadIdx.x * kEach + i];
  uint64_t at = block_scan(mine, s.warp_sum, total) - mine;
  need = min(need, total);
  if (threadIdx.x == 0 && to > total) s.bin_to = kEach * kThreads - 1;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (need > at && need <= at + w[i]) {
      s.bin_at = threadIdx.x * kEach + i;
      s.need = need - at;
    }
    if (to > at && to <= at + w[i]) s.bin_to = threadIdx.x * kEach + i;
    at += w[i];
  }
  __syncthreads();
  bin = s.bin_at;
  last = s.bin_to;
  need = s.need;
}

// What is looked for in a list of keys: the key at which the sum of masses, from the largest key on, reaches
//   count: `whole`      share: x of `whole` (0: of the list's mass)      draw: more than x of the list's
// Where the list's sum does not reach it, and `all` does not say that there is nothing else: none.
enum class Mode { count, share, draw };
struct Want {
  Mode mode;
  double x;
  uint64_t whole;
  bool all;
  __device__ __forceinline__ uint64_t of(uint64_t total) const {
    if (total == 0) return 0;
    if (mode == Mode::draw) return min((uint64_t)(x * (double)total), total - 1) + 1;
    uint64_t n = whole;
    if (mode == Mode::share) {
      const double need = ceil(fmax(x, 0.0) * (double)(whole ? whole : total));
      n = need >= 1.0 ? (uint64_t)need : 1;
    }
    return n <= total ? n : all ? total : 0;
  }
};

// That key, among the keys from `low` on with masses of `least` and up (masses null: of 1 each), and its mass in
// s.border_mass; 0 if there is none. Drawn is in the order of the ids: a key's halves are exchanged for that, and
// so are those of the result. The keys are cut into bins by their distance from `high` (the range is looked up
// where high is below `end`), the one with the border again, until it has few, which are compared.
// (One function for all three, which a row calls in turn: it is bound by its code's way to the SM.)
__device__ __noinline__ uint64_t pick(Scratch &s, const uint64_t *keys, const uint64_t *masses, int n, uint64_t low, uint64_t least, uint64_t high,
                                      uint64_t end, const Want want) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool turned = want.mode == Mode::draw;
  if (high < end && n > kFew) {
    uint64_t from = ~0ull, to = 0;
    for (int i = tid; i < n; i += kThreads) {
      from = min(from, keys[i]);
      to = max(to, keys[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      from = min(from, __shfl_xor_sync(0xffffffffu, from, o));
      to = max(to, __shfl_xor_sync(0xffffffffu, to, o));
    }
    if (lane == 0) {
      s.range[0][warp] = from;
      s.range[1][warp] = to;
    }
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) {
      from = min(from, s.range[0][i]);
      to = max(to, s.range[1][i]);
    }
    high = to;
    end = from;
  }
  uint64_t need = 0;
  if (n <= kFew) {
    __syncthreads();  // (what was in the keys' place is read)
    if (tid == 0) s.count = 0;
    __syncthreads();
    uint64_t w = 0, total;
    if (tid < n && keys[tid] >= low) {
      w = masses ? masses[tid] : 1;
      if (w < least) w = 0;
      if (w > 0) {
        const uint32_t to = atomicAdd(&s.count, 1u);
        s.few[to] = turned ? (keys[tid] << 32) | (keys[tid] >> 32) : keys[tid];
        s.few_mass[to] = w;
      }
    }
    block_scan(w, s.warp_sum, total);
    need = want.of(total);
    if (tid == 0) s.total = total;
    if (need == 0) return 0;
  } else for (bool first = true;; first = false) {
    const int shift = max(0, 64 - __clzll((long long)((high - end) | 1)) - 11);
    __syncthreads();  // (what was in the bins' place is read)
#pragma unroll 4
    for (int i = tid; i < kBins * 3; i += kThreads) (&s.limb[0][0])[i] = 0;
    if (tid == 0) s.count = 0;
    __syncthreads();
    auto at = [&](int i, uint64_t &pos, uint64_t &w) -> bool {
      const uint64_t key = keys[i];
      w = masses ? masses[i] : 1;
      pos = turned ? (key << 32) | (key >> 32) : key;
      return key >= low && w >= least && pos <= high && pos >= end;
    };
    uint64_t pos, w;
#pragma unroll 1
    for (int i = tid; i < n; i += kThreads)
      if (at(i, pos, w)) add_mass(s.limb, (uint32_t)((high - pos) >> shift), w);
    __syncthreads();
    constexpr int kEach = kBins / kThreads;
    uint64_t mine[kEach], sum = 0, total;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int b = tid * kEach + i;
      sum += mine[i] = s.limb[0][b] + ((uint64_t)s.limb[1][b] << kLimb) + ((uint64_t)s.limb[2][b] << (2 * kLimb));
    }
    uint64_t run = block_scan(sum, s.warp_sum, total) - sum;
    if (first) {
      need = want.of(total);
      if (tid == 0) s.total = total;
    }
    if (need == 0) return 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (need > run && need <= run + mine[i]) {
        s.bin_at = tid * kEach + i;
        s.need = need - run;
      }
      run += mine[i];
    }
    __syncthreads();
    const uint32_t bin = s.bin_at;
    need = s.need;
#pragma unroll 1
    for (int i = tid; i < n; i += kThreads)
      if (at(i, pos, w) && (uint32_t)((high - pos) >> shift) == bin) {
        const uint32_t to = atomicAdd(&s.count, 1u);
        if (to < (uint32_t)kFew) {
          s.few[to] = pos;
          s.few_mass[to] = w;
        }
      }
    __syncthreads();
    if (s.count <= (uint32_t)kFew) break;
    high -= (uint64_t)bin << shift;
    end = max(end, high - (((uint64_t)1 << shift) - 1));
  }
  // few: what is at or ahead of a key is added up, by some neighbouring threads a key
  const int few = (int)s.count;
  int parts = 1;
  while (parts < 32 && 2 * parts * few <= kThreads) parts *= 2;
  const int at = tid / parts;
  const uint64_t key = at < few ? s.few[at] : ~0ull;
  uint64_t run = 0;
  for (int i = tid & (parts - 1); i < few; i += parts) run += s.few[i] >= key ? s.few_mass[i] : 0;
  for (int o = parts >> 1; o > 0; o >>= 1) run += __shfl_xor_sync(0xffffffffu, run, o);
  if (at < few && run >= need && run - s.few_mass[at] < need) {
    s.border = key;
    s.border_mass = s.few_mass[at];
  }
  __syncthreads();
  return s.border;
}

// The masses of all CTAs' warps (s.kept) together, and what is ahead of this warp's.
__device__ __forceinline__ uint64_t cluster_sum(Shared &s, uint64_t &before) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  __syncthreads();
  if (threadIdx.x < ctas) {
    uint64_t whole = 0;
    for (int i = 0; i < kWarps; ++i) whole += s.kept[i];
    cluster.map_shared_rank(s.cta_sum, threadIdx.x)[rank] = whole;
  }
  cluster.sync();
  uint64_t total = 0;
  before = 0;
  for (int i = 0; i < ctas; ++i) {
    total += s.cta_sum[i];
    if (i < rank) before += s.cta_sum[i];
  }
  for (int i = 0; i < (int)threadIdx.x >> 5; ++i) before += s.kept[i];
  return total;
}

// The border of the shortest beginning of the order (of the keys from `above` on) whose mass, or whose number,
// reaches `need`: the key of its last member. MASS: they have the mass `whole` together; s.kept becomes the
// warps' masses from the border on, or `summed` false.
template <bool MASS>
__device__ __noinline__ uint64_t find_border(Shared &s, const Columns columns, const Row row, float t, float per_logit,
                                             uint64_t above, uint64_t whole, uint64_t need, bool &summed) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5;
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  Span span;
  span.low = above;
  span.high = ~0ull;
  span.shift = -1;
  span.top = row.top;
  span.per_logit = per_logit;
  for (;;) {
    const bool first = span.shift < 0;
    __syncthreads();  // (what was in the bins' place is read)
    for (int i = tid; i < (first ? kFirst : kBins * (MASS ? 3 : 1)); i += kThreads) (&s.limb[0][0])[i] = 0;
    __syncthreads();
    if (!first) key_bins<MASS>(columns, span, row, s.table, s.limb);
    else if (MASS && above) share_bins<true>(columns, span, 2.0f * 1.44269504f / t, 0x1p75f / (float)whole, s.first);
    else if (MASS) share_bins<false>(columns, span, 2.0f * 1.44269504f / t, 0x1p75f / (float)whole, s.first);
    else count_bins(columns, span, s.first);
    if (!first) join_limbs<MASS>(s);
    cluster.sync();
    // every CTA adds up a share of the bins and gives it to all: `parts` threads a bin, some CTAs each
    {
      const int per = kBins / ctas, parts = max(1, kThreads / per), each = ctas / min(parts, ctas);
      const int b0 = tid % min(per, kThreads), part = tid / min(per, kThreads);
      for (int b = b0; b < per; b += kThreads) {
        uint64_t x[4] = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r < each && part * each + r < ctas) x[r] = cluster.map_shared_rank(s.bin, part * each + r)[rank * per + b];
        uint64_t sum = (x[0] + x[1]) + (x[2] + x[3]);
        if (parts > 1) {
          s.part[tid] = sum;
          __syncthreads();
          sum = 0;
          for (int i = 0; i < parts; ++i) sum += s.part[i * per + b];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r < each && part * each + r < ctas) cluster.map_shared_rank(s.whole, part * each + r)[rank * per + b] = sum;
      }
    }
    cluster.sync();
    uint32_t bin, last;
    if (MASS && first) {
      // shares are off by 1/2 each, and by 2^-17 where e^x is made in f32: 46 powers of 2 at most with three
      // roundings of 2^-24, and the instruction's 2^-22. The border lies in the bins between.
      const double aim = (double)need * (0x1p31 / (double)whole), off = 0.5 * columns.share * ctas + 0x1p15;
      uint64_t from = aim - off > 1.0 ? (uint64_t)(aim - off) : 1;
      find_bin<true>(s, s.whole, from, (uint64_t)(aim + off) + 2, bin, last);
      if (t < 1e-30f || t > 1e30f) bin = 0, last = kFirst - 1;  // (e^x in f32 may be anything)
    } else {
      if (first) find_bin<true>(s, s.whole, need, 0, bin, last);
      else find_bin<false>(s, s.whole, need, 0, bin, last);
      last = bin;
    }
    // the bins' keys: of each CTA, then of all in every one
    if (tid == 0) s.count = 0;
    __syncthreads();
    uint64_t ahead = 0;
    if (first && MASS && above) ahead = collect<true, MASS, MASS>(columns, span, row, s.table, bin, last, s.list, &s.count);
    else if (first) ahead = collect<true, MASS, false>(columns, span, row, s.table, bin, last, s.list, &s.count);
    else collect<false, false, true>(columns, span, row, s.table, bin, bin, s.list, &s.count);
    if (MASS && first) {
      ahead = warp_sum(ahead);
      if ((tid & 31) == 0) s.kept[warp] = ahead;
    }
    __syncthreads();
    if (tid < ctas) {
      uint64_t sum = 0;
      if (MASS && first)
        for (int i = 0; i < kWarps; ++i) sum += s.kept[i];
      cluster.map_shared_rank(s.cta_sum, tid)[rank] = sum;
      cluster.map_shared_rank(s.cta_count, tid)[rank] = s.count;
    }
    cluster.sync();
    uint32_t n = 0, at = 0;
    uint64_t sum = 0;
    for (int i = 0; i < ctas; ++i) {
      if (i == rank) at = n;
      n += s.cta_count[i];
      sum += s.cta_sum[i];
    }
    if (MASS && first) need = need > sum ? need - sum : 1;
    if (n <= (uint32_t)kList)
      for (int i = tid; i < (int)s.count * ctas; i += kThreads)
        cluster.map_shared_rank(s.whole, i & (ctas - 1))[at + i / ctas] = s.list[i / ctas];
    cluster.sync();
    if (n <= (uint32_t)kList) {
      if (MASS)
        for (int i = tid; i < (int)n; i += kThreads) s.masses[i] = mass_of_key(s.table, row, s.whole[i]);
      __syncthreads();
      const uint64_t border = pick(s, s.whole, MASS ? s.masses : nullptr, (int)n, 0, 0, 0, 1, Want{Mode::count, 0.0, need, true});
      if (MASS && first) {
        summed = true;
        for (int i = tid; i < (int)n; i += kThreads) {
          const uint32_t id = ~(uint32_t)s.whole[i] - (uint32_t)(rank * columns.share);
          if (s.whole[i] >= border && id < (uint32_t)columns.share)
            atomicAdd(&s.kept[id / (uint32_t)(columns.n * 128)], (unsigned long long)s.masses[i]);
        }
        __syncthreads();  // (a caller may write the sums anew)
      }
      return border;
    }
    // too many: their range, from the few that are listed and the bin's own
    if (first) {
      // the smallest and the largest key whose bin it is
      uint64_t lo = ~0ull, hi = 0;
      for (int i = 0; i < columns.n; ++i) {
        const float4 x = columns.at(i);
        const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t id = columns.id + i * 128 + k;
          if (span.first_bin(v[k]) < bin || span.first_bin(v[k]) > last || !span.has(v[k], id)) continue;
          lo = min(lo, rank_key(v[k], id));
          hi = max(hi, rank_key(v[k], id));
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      if ((tid & 31) == 0) {
        s.range[0][warp] = lo;
        s.range[1][warp] = hi;
      }
      __syncthreads();
      for (int i = 0; i < kWarps; ++i) {
        lo = min(lo, s.range[0][i]);
        hi = max(hi, s.range[1][i]);
      }
      if (tid < ctas) {
        cluster.map_shared_rank(s.whole, tid)[2 * rank] = lo;
        cluster.map_shared_rank(s.whole, tid)[2 * rank + 1] = hi;
      }
      cluster.sync();
      for (int r = 0; r < ctas; ++r) {
        lo = min(lo, s.whole[2 * r]);
        hi = max(hi, s.whole[2 * r + 1]);
      }
      span.high = hi;
      span.low = lo;
      span.shift = max(0, 64 - __clzll((long long)(hi - lo)) - 11);
      cluster.sync();  // (before the bins of the next round are written there)
    } else {
      // the bin's own range of keys
      span.high -= (uint64_t)bin << span.shift;
      span.low = max(span.low, span.high - (((uint64_t)1 << span.shift) - 1));
      span.shift = max(0, span.shift - 11);
    }
  }
}

// What the options leave: logits from a border on (BORDER: there is one), of a mass of `least` and up. A lane's four
// masses, as 2^52 plus each; false where the whole warp has none.
struct Kept {
  float v;
  uint32_t id;
  double least;
  template <bool BORDER>
  __device__ __forceinline__ bool masses(const float4 x, uint32_t at, const Row &row, const double *table, double (&m)[4]) const {
    float l[4] = {x.x, x.y, x.z, x.w};
    if (BORDER) {
      bool any = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (!from_on(l[k], at + k, v, id)) l[k] = -INFINITY;
        any |= l[k] > -INFINITY;
      }
      if (!__any_sync(0xffffffffu, any)) return false;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = rounded_mass(table, row, l[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = m[k] >= least ? m[k] : kWhole;
    if (row.far)
#pragma unroll
      for (int k = 0; k < 4; ++k) m[k] = l[k] > -INFINITY ? m[k] : kWhole;
    return true;
  }
};
template <bool BORDER>
__device__ __noinline__ uint64_t sum_kept(const Columns c, const Kept kept, const Row row, const double *table) {
  uint64_t sum = 0;
  Stream next(c);
#pragma unroll 1
  for (int i = 0; i < c.n; ++i) {
    double m[4];
    if (kept.masses<BORDER>(next.take(i), c.id + i * 128, row, table, m))
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += bits_of(m[k]) - kWholeBits;
  }
  return sum;
}

__device__ __forceinline__ uint64_t block_sum(Scratch &s, uint64_t v) {
  uint64_t total;
  block_scan(v, s.warp_sum, total);
  return total;
}

__device__ __forceinline__ double next_f64(uint64_t z) {  // of the advanced state
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
  z ^= z >> 31;
  return (double)(z >> 11) / (double)(1ull << 53);
}
constexpr uint64_t kStep = 0x9e3779b97f4a7c15ull;

// A row's options. (All are loaded whatever the others are: their latencies overlap.)
struct Options {
  bool greedy;
  int k;  // 0: all
  float p, t, low_p;
};
__device__ __forceinline__ Options options_of(const Args &a, int64_t r) {
  Options o;
  o.t = a.temperature ? a.temperature[r] : 1.0f;
  o.k = a.top_k ? a.top_k[r] : 0;
  o.p = a.top_p ? a.top_p[r] : 1.0f;
  o.low_p = a.min_p ? a.min_p[r] : 0.0f;
  o.greedy = !(o.t > 0.0f);
  if (o.k < 0 || o.k >= a.vocab) o.k = 0;
  if (o.greedy) {
    o.k = 0;
    o.p = 1.0f;
    o.t = o.low_p = 0.0f;
  }
  return o;
}

// ---- first launch: a CTA a piece of a row. Its largest logit; where all of the row counts, its sum of
// masses, relative to its own largest; and its largest keys, those from the q-th largest thread's largest on.
__global__ void __launch_bounds__(kSurvey) survey_kernel(const Args a) {
  extern __shared__ __align__(16) float4 vals4[];  // [piece / 4], thread t's at t, t + kSurvey, ...
  __shared__ double table[kTable];
  __shared__ uint32_t bins[kSurvey];
  __shared__ float tops[kSurvey / 32], bottoms[kSurvey / 32];
  __shared__ uint32_t counts[kSurvey / 32], border, given;
  __shared__ uint64_t sums[kSurvey / 32];
  __shared__ __align__(8) uint64_t arrived;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / a.pieces;
  const int piece = blockIdx.x - (int)r * a.pieces;
  if (tid < kTable) table[tid] = kPowers[tid];
  bins[tid] = 0;
  if (tid == 0) {
    given = 0;
    gqd::mbar_init(&arrived, 1);
    gqd::fence_mbar_init();
  }
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  if (blockIdx.x == 0 && tid < 2) a.n_todo[tid] = 0;
  const int id0 = piece * a.piece, n = min(a.vocab - id0, a.piece);
  const float *from = a.logits + r * a.ld + id0;
  const Options o = options_of(a, r);
  const bool greedy = o.greedy;
  const int k = o.k;
  const float p = o.p, t = o.t;
  const bool sum_all = !greedy && k == 0 && (p < 1.0f || !(o.low_p > 0.0f));
  const int steps = a.piece / (4 * kSurvey);
  // the piece as one copy: all of an SM's pieces are on their way at once (loads by the threads: 91 us for the
  // mixed options, this way 85; a top_k of 64 37 and 29)
  if (a.wide && n % 4 == 0) {
    if (tid == 0) {
      gqd::mbar_arrive_expect_tx(&arrived, (uint32_t)n * 4);
      gqd::bulk_g2s(vals4, from, (uint32_t)n * 4, &arrived);
    }
    for (int i = n / 4 + tid; i < a.piece / 4; i += kSurvey) vals4[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    __syncthreads();  // (the barrier is made)
    if (!__syncthreads_and(gqd::mbar_wait_bounded(&arrived, 0))) {
      // a copy that does not come: an error, and a piece without a token
      if (tid == 0) {
        gqd::report(a.err, GQ_DEVERR_WAIT_TIMEOUT);
        (void)gqd::mbar_wait_bounded(&arrived, 0, 100000000ull);
        const int64_t at = r * a.pieces + piece;
        a.piece_top[at] = -INFINITY;
        a.piece_from[at] = -INFINITY;
        a.piece_given[at] = 0;
        a.piece_mass[at] = 0;
      }
      return;
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < steps; ++i) vals4[tid + i * kSurvey] = raw_logits(from, 4 * (tid + i * kSurvey), n, a.wide);
  }
  float top = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < steps; ++i) {
    const float4 v = vals4[tid + i * kSurvey];  // (its own, or what has arrived)
    top = fmaxf(top, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
  }
  top += 0.0f;  // (0 for -0; a NaN is no maximum)
  const float mine = top;
  float bottom = mine > -INFINITY ? mine : INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bottom = fminf(bottom, __shfl_xor_sync(0xffffffffu, bottom, o));
  }
  if (lane == 0) {
    tops[warp] = top;
    bottoms[warp] = bottom;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSurvey / 32; ++i) {
    top = fmaxf(top, tops[i]);
    bottom = fminf(bottom, bottoms[i]);
  }
  // the q-th largest of the threads' largest, by its bin
  // (a piece has k / pieces of the row's k largest, give or take: twice that and 12 leave one row in a million
  // of independent logits to the last launch; and a thread's largest stands for others of its own, which need room)
  const int q = min((k > 0 ? 2 * min(k, kGiven) : kGiven) / a.pieces + 12, min(kSurvey / 2, a.give * 3 / 4));
  const float per = (float)(kSurvey - 1) / (top - bottom);
  const uint32_t b = __float_as_uint(fminf((top - mine) * per, (float)(kSurvey - 1)) + 8388608.0f) & (kSurvey - 1);
  if (mine > -INFINITY) atomicAdd(&bins[b], 1u);
  __syncthreads();
  uint32_t run = bins[tid];
  const uint32_t own = run;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) counts[warp] = run;
  __syncthreads();
  uint32_t lanes = 0;
#pragma unroll
  for (int i = 0; i < kSurvey / 32; ++i) {
    if (i < warp) run += counts[i];
    lanes += counts[i];
  }
  if (run >= (uint32_t)q && run - own < (uint32_t)q) border = tid;
  __syncthreads();
  float least = mine > -INFINITY && lanes >= (uint32_t)q && b <= border ? mine : INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  if (lane == 0) bottoms[warp] = least;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSurvey / 32; ++i) least = fminf(least, bottoms[i]);
  if (lanes < (uint32_t)q) least = -INFINITY;  // (all that there are)
  uint64_t all = 0;
  if (sum_all && top > -INFINITY && top < INFINITY) {  // (infinities: the last launch)
    const Row row = row_of(top, t);
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      const float4 x = vals4[tid + i * kSurvey];
      const float v[4] = {x.x, x.y, x.z, x.w};
      double m[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) m[j] = rounded_mass(table, row, v[j]);
      if (row.far)
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = v[j] > -INFINITY ? m[j] : kWhole;
#pragma unroll
      for (int j = 0; j < 4; ++j) all += bits_of(m[j]) - kWholeBits;
    }
    all = warp_sum(all);
  }
  __syncwarp();
  // the keys: a lane marks its own, a warp takes places for all of them
  const float from_there = fmaxf(least, -3.402823466e+38f);  // (-inf is not given)
  if (__any_sync(0xffffffffu, mine >= from_there)) {
    uint32_t mark = 0;
    for (int i = 0; i < steps; ++i) {
      const float4 x = vals4[tid + i * kSurvey];
      mark |= (uint32_t)((x.x >= from_there) | (x.y >= from_there) << 1 | (x.z >= from_there) << 2 | (x.w >= from_there) << 3) << (4 * i);
    }
    uint32_t to = __popc(mark);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= o) to += up;
    }
    uint32_t from0 = 0;
    if (lane == 31) from0 = atomicAdd(&given, to);
    to += __shfl_sync(0xffffffffu, from0, 31) - __popc(mark);
    uint64_t *keys = a.piece_keys + ((int64_t)r * a.pieces + piece) * a.give;
    for (; mark && to < (uint32_t)a.give; mark &= mark - 1, ++to) {
      const int i = __ffs(mark) - 1, c = 4 * (tid + (i >> 2) * kSurvey) + (i & 3);
      keys[to] = rank_key(reinterpret_cast<const float *>(vals4)[c] + 0.0f, id0 + c);
    }
  }
  if (lane == 0) sums[warp] = all;
  __syncthreads();
  if (tid == 0) {
    all = 0;
    for (int i = 0; i < kSurvey / 32; ++i) all += sums[i];
    const int64_t at = (int64_t)r * a.pieces + piece;
    a.piece_top[at] = top;
    a.piece_from[at] = given > (uint32_t)a.give ? INFINITY : least;  // (from there on all are given: not more than there is room for)
    a.piece_given[at] = (int)min(given, (uint32_t)a.give);
    a.piece_mass[at] = all;
  }
}

// ---- second launch: a CTA a row, from what was found in its pieces. Rows that it cannot be sure of are left to
// the last launch: a border below what all pieces have given, infinities.
__global__ void __launch_bounds__(kThreads) finish_kernel(const Args a) {
  __shared__ Scratch s;
  extern __shared__ __align__(16) uint64_t keys[];  // [kMostGiven], and their masses
  uint64_t *masses = keys + kMostGiven;
  __shared__ int starts[kMaxPieces + 1];
  __shared__ double piece_sum[kMaxPieces], warp_d[kWarps];
  __shared__ float tops[kWarps], froms[kWarps];
  __shared__ int n_keys, chosen;
  __shared__ double rest;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x;
  if (tid < kTable) s.table[tid] = kPowers[tid];
  if (tid == 0) {
    n_keys = 0;
    chosen = -1;
  }
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  // all that may be needed is loaded at once
  const Options o = options_of(a, r);
  const uint64_t state = a.rng ? a.rng[r] : 0;
  const double given_u = a.rng ? 0.0 : a.uniforms[r];
  const int64_t at0 = r * a.pieces;
  // (kMaxPieces <= kThreads: a thread a piece)
  const bool has = tid < a.pieces;
  const float my_top = has ? a.piece_top[at0 + tid] : -INFINITY;
  const int my_n = has ? a.piece_given[at0 + tid] : 0;
  const uint64_t my_mass = has ? a.piece_mass[at0 + tid] : 0;
  float top = my_top, from = has ? a.piece_from[at0 + tid] : -INFINITY;
  uint64_t some[kMostGiven / kThreads];
#pragma unroll
  for (int i = 0; i < kMostGiven / kThreads; ++i)
    some[i] = tid + i * kThreads < a.pieces * a.give ? a.piece_keys[at0 * a.give + tid + i * kThreads] : 0;
  const bool greedy = o.greedy;
  const int k = o.k;
  const float p = o.p, t = o.t, low_p = o.low_p;
  double u = 0.0;
  if (!greedy) {
    u = a.rng ? next_f64(state + kStep) : given_u;
    u = u >= 0.0 ? fmin(u, 1.0 - 0x1p-53) : 0.0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    from = fmaxf(from, __shfl_xor_sync(0xffffffffu, from, o));
  }
  if (lane == 0) {
    tops[warp] = top;
    froms[warp] = from;
  }
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) {
    top = fmaxf(top, tops[i]);
    from = fmaxf(from, froms[i]);  // from there on the pieces have given all
  }
  if (tid == 0) {
    a.drawn[r] = u;
    if (a.rng && !greedy) a.rng[r] = state + kStep;
    if (top == INFINITY) a.todo[atomicAdd(a.n_todo, 1)] = (int)r;
    if (top == -INFINITY) {  // nothing that can be drawn
      a.tokens[r] = -1;
      if (a.probs) a.probs[r] = 0.0f;
    }
  }
  if (top == INFINITY || top == -INFINITY) return;
  const Row row = row_of(top, t);
  uint64_t least = 1;
  if (low_p > 0.0f) least = max(least, (uint64_t)ceil(fmin((double)low_p, 1.0) * (double)(1ull << kOne)));

  if (!greedy && k == 0 && !(p < 1.0f) && !(low_p > 0.0f)) {
    // all tokens: the piece in which the sum passes u times the whole, and the token in it
    double mass = 0.0;
    if (my_top > -INFINITY) mass = (double)my_mass * exp(((double)my_top - (double)top) / (double)t);
    double run = mass;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (lane == 31) warp_d[warp] = run;
    __syncthreads();
    double total = 0.0, before = 0.0;
    for (int i = 0; i < kWarps; ++i) {
      if (i == warp) before = total;
      total += warp_d[i];
    }
    run += before;
    const double want = u * total;
    if (has) piece_sum[tid] = run;
    // (roundings may leave the end of the last piece short of the whole: the last piece that has any takes it)
    if (mass > 0.0 && run > want) atomicMin(reinterpret_cast<unsigned int *>(&chosen), (unsigned int)tid);
    __syncthreads();
    if (chosen < 0 && mass > 0.0) atomicMax(&n_keys, tid);
    __syncthreads();
    const int piece = chosen >= 0 ? chosen : n_keys;
    if (tid == piece) rest = fmax(want - (piece > 0 ? piece_sum[piece - 1] : 0.0), 0.0) / exp(((double)my_top - (double)top) / (double)t);
    __syncthreads();
    const float piece_top = a.piece_top[at0 + piece];
    const uint64_t whole = a.piece_mass[at0 + piece];
    const uint64_t aim = min((uint64_t)rest, whole - 1);
    const Row prow = row_of(piece_top, t);
    const int id0 = piece * a.piece, n = min(a.vocab - id0, a.piece);
    const float *vals = a.logits + r * a.ld + id0;
    // a warp a run of columns
    const int each = a.piece / kWarps;
    auto mass_at = [&](int c) -> uint64_t {
      if (c >= n) return 0;
      const float v = fmaxf(vals[c], -INFINITY) + 0.0f;
      return mass_of(s.table, prow, v);
    };
    uint64_t sum = 0;
#pragma unroll 4
    for (int c = warp * each + lane; c < (warp + 1) * each; c += 32) sum += mass_at(c);
    sum = warp_sum(sum);
    if (lane == 0) s.warp_sum[warp] = sum;
    __syncthreads();
    uint64_t ahead = 0;
    for (int i = 0; i < warp; ++i) ahead += s.warp_sum[i];
    if (aim < ahead || aim >= ahead + sum) return;
    for (int c = warp * each + lane; c < (warp + 1) * each; c += 32) {
      const uint64_t w = mass_at(c), incl = warp_scan(w) + ahead;
      const uint32_t past = __ballot_sync(0xffffffffu, incl > aim);
      if (past) {
        if (lane == __ffs(past) - 1) {
          a.tokens[r] = id0 + c;
          if (a.probs) a.probs[r] = (float)((double)w * exp(((double)piece_top - (double)top) / (double)t) / total);
        }
        return;
      }
      ahead = __shfl_sync(0xffffffffu, incl, 31);
    }
    return;
  }

  // the keys that were given, together
  {
    uint64_t total;
    const uint64_t ends = block_scan((uint64_t)my_n, s.warp_sum, total);
    if (has) starts[tid + 1] = (int)ends;
    if (tid == 0) starts[0] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMostGiven / kThreads; ++i) {
      const int at = tid + i * kThreads, piece = at / a.give, j = at - piece * a.give;
      if (piece < a.pieces && j < starts[piece + 1] - starts[piece]) keys[starts[piece] + j] = some[i];
    }
    __syncthreads();
  }
  const int n = starts[a.pieces];
#pragma unroll 1
  for (int i = tid; i < n; i += kThreads) masses[i] = mass_of_key(s.table, row, keys[i]);
  __syncthreads();
  const uint64_t end = (uint64_t)key_of(from) << 32, high = rank_key(top, 0);  // from `end` on the list has all
  const bool all = from == -INFINITY;
  uint64_t whole = 0;  // (0: of the list)
  if (k == 0 && p < 1.0f) {
    const double f = my_top > -INFINITY ? exp(((double)my_top - (double)top) / (double)t) : 0.0;
    whole = block_sum(s, has ? (uint64_t)((double)my_mass * f) : 0);
    if (tid == 0) a.row_mass[r] = whole;
  }
  bool known = from <= top;
  uint64_t border = end;
  if (greedy) {
    border = (uint64_t)key_of(top) << 32;
  } else if (known) {
    if (k > 0) known = (border = pick(s, keys, nullptr, n, end, 0, high, end, Want{Mode::count, 0.0, (uint64_t)k, all})) != 0;
    if (known && p < 1.0f)
      known = (border = pick(s, keys, masses, n, border, 0, high, border, Want{Mode::share, (double)p, whole, false})) != 0;
    // min_p alone: what is not in the list must be below it
    if (known && k == 0 && !(p < 1.0f) && !all && mass_of_key(s.table, row, end) >= least) known = false;
  }
  if (!known) {
    if (tid == 0) a.todo[atomicAdd(a.n_todo, 1)] = (int)r;
    return;
  }
  const uint64_t drawn = pick(s, keys, masses, n, border, least, ~0ull << 32 | ~0u, (uint64_t)~(uint32_t)a.vocab << 32, Want{Mode::draw, u, 0, true});
  if (tid == 0) {
    a.tokens[r] = (int32_t)~(uint32_t)(drawn >> 32);
    if (a.probs) a.probs[r] = greedy ? 1.0f : (float)((double)s.border_mass / (double)s.total);
  }
}

// ---- last launch: a cluster a row, whatever the options leave.
__device__ __forceinline__ void sample_row(const Args &a, Shared &s, int64_t r) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster.block_rank();
  const Options o = options_of(a, r);
  const bool greedy = o.greedy;
  const int k = o.k;
  const float p = o.p, t = o.t, low_p = o.low_p;
  const double u = a.drawn[r];
  // the row's largest, and the smallest from which on a piece has given its keys
  float top = tid < a.pieces ? a.piece_top[r * a.pieces + tid] : -INFINITY;
  float from = tid < a.pieces ? a.piece_from[r * a.pieces + tid] : INFINITY;
  if (from == -INFINITY) from = INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    from = fminf(from, __shfl_xor_sync(0xffffffffu, from, o));
  }
  if (lane == 0) {
    s.warp_top[warp] = top;
    s.warp_from[warp] = from;
  }
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) {
    top = fmaxf(top, s.warp_top[i]);
    from = fminf(from, s.warp_from[i]);
  }
  const bool infinite = top == INFINITY;
  if (infinite) top = 0.0f;
  const int id0 = rank * a.share;
  const Columns columns{a.logits + r * a.ld, a.run / 128, min(id0 + a.share, a.vocab), a.share, (uint32_t)(id0 + warp * a.run + lane * 4), a.wide != 0, infinite};
  // bins over some times the span of the keys that were given, for masses over those that have any: what lies
  // below is one bin, which another round can cut
  const float span = from < top && !infinite ? 4.0f * (top - from) : 64.0f, heavy = 32.0f * t;
  const Row row = row_of(top, t);
  uint64_t above = 0, before;
  double least = kWhole + 1.0;
  bool summed = false;  // s.kept is the warps' masses that are kept
  auto sum_of = [&](uint64_t border) {
    const Kept kept{logit_of(border), ~(uint32_t)border, least};
    uint64_t sum = 0;
    if (top > -INFINITY) sum = border ? sum_kept<true>(columns, kept, row, s.table) : sum_kept<false>(columns, kept, row, s.table);
    sum = warp_sum(sum);
    if (lane == 0) s.kept[warp] = sum;
  };
  if (!greedy && top > -INFINITY) {
    if (k > 0)
      above = find_border<false>(s, columns, row, t, (float)(kFirst - 1) / span, 0, 0, (uint64_t)k, summed);
    if (p < 1.0f) {
      uint64_t whole;
      if (k == 0 && !infinite) {
        whole = a.row_mass[r];
      } else {
        sum_of(above);
        whole = cluster_sum(s, before);
        cluster.sync();  // (before the sums are written again)
      }
      const double want = ceil(fmax((double)p, 0.0) * (double)whole);
      above = find_border<true>(s, columns, row, t, (float)(kFirst - 1) / fminf(span, heavy), above, whole,
                                min(want >= 1.0 ? (uint64_t)want : (uint64_t)1, whole), summed);
    }
    if (low_p > 0.0f) {
      least = fmax(least, kWhole + ceil(fmin((double)low_p, 1.0) * (double)(1ull << kOne)));
      summed = false;
    }
  }
  if (!summed) sum_of(above);
  const Kept kept{above ? logit_of(above) : -INFINITY, above ? ~(uint32_t)above : ~0u, least};
  const uint64_t total = cluster_sum(s, before);
  uint64_t at = (uint64_t)(u * (double)total);
  if (total > 0) at = min(at, total - 1);
  if (at < before || at >= before + s.kept[warp]) return;
  // the warp in whose run the sum passes `at`
  for (int i = 0; i < columns.n; ++i) {
    double m[4];
    uint64_t w[4] = {0, 0, 0, 0};
    const uint32_t at_id = columns.id + i * 128;
    if (!kept.masses<true>(columns.at(i), at_id, row, s.table, m)) continue;
    for (int k = 0; k < 4; ++k) w[k] = (uint64_t)(m[k] - kWhole);
    const uint64_t four = (w[0] + w[1]) + (w[2] + w[3]);
    const uint64_t incl = warp_scan(four) + before;
    const uint32_t past = __ballot_sync(0xffffffffu, incl > at);
    if (past) {
      if (lane == __ffs(past) - 1) {
        uint64_t run = incl - four;
        for (int k = 0; k < 4; ++k) {
          run += w[k];
          if (run > at) {
            a.tokens[r] = (int32_t)(columns.id + i * 128 + k);
            if (a.probs) a.probs[r] = greedy ? 1.0f : (float)((double)w[k] / (double)total);
            break;
          }
        }
      }
      return;
    }
    before = __shfl_sync(0xffffffffu, incl, 31);
  }
}

__global__ void __launch_bounds__(kThreads, 1) sample_requests_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t of_cta[];
  Shared &s = *reinterpret_cast<Shared *>(of_cta);
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks();
  if (threadIdx.x < kTable) s.table[threadIdx.x] = kPowers[threadIdx.x];
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const int n = *a.n_todo;
  if (n == 0) return;
  // a cluster takes the next row that is left, until there is none
  for (;;) {
    cluster.sync();  // (all have begun, and are done with the row before)
    if (threadIdx.x == 0 && cluster.block_rank() == 0) {
      const int i = atomicAdd(a.n_todo + 1, 1);
      for (int c = 0; c < ctas; ++c) *cluster.map_shared_rank(&s.turn, c) = i;
    }
    cluster.sync();
    if (s.turn >= n) return;
    sample_row(a, s, a.todo[s.turn]);
  }
}

}  // namespace

extern "C" int gq_sample_requests(gq_ctx *ctx, const float *logits, int64_t m, int64_t vocab, int64_t ld, const float *temperature,
                                  const int32_t *top_k, const float *top_p, const float *min_p, const double *uniforms,
                                  uint64_t *rng_state, int32_t *tokens, float *probs) {
  if (!ctx) return GQ_ERR_INVALID_ARGUMENT;
  const int rc = gq_enter_ctx(ctx);
  if (rc != GQ_OK) return rc;
  if (ld == 0) ld = vocab;
  if (m < 0 || vocab < 1 || ld < vocab) return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "sample_requests: bad m, vocab or ld");
  if (vocab > kMaxVocab || m > INT32_MAX / kMaxCluster)
    return gq_fail(ctx, GQ_ERR_UNSUPPORTED, "sample_requests: vocab above 524288, or too many rows");
  if (m == 0) return GQ_OK;
  if (!logits || !tokens) return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "sample_requests: null pointer");
  if (!uniforms == !rng_state)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "sample_requests: either uniforms or rng_state, one of them");
  Args a{};
  a.logits = logits;
  a.ld = ld;
  a.vocab = (int)vocab;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.uniforms = uniforms;
  a.rng = rng_state;
  a.tokens = tokens;
  a.probs = probs;
  a.err = ctx->dev_err;
  a.wide = (uintptr_t)logits % 16 == 0 && ld % 4 == 0;
  // pieces of a row: as large as leaves two for every SM
  a.piece = kMaxPiece;
  const int64_t together = std::min<int64_t>(m, kRows);
  auto pieces = [&](int piece) { return (vocab + piece - 1) / piece; };
  while (a.piece > 2048 && together * pieces(a.piece) < 2 * (int64_t)ctx->num_sms && pieces(a.piece / 2) <= kMaxPieces) a.piece /= 2;
  a.pieces = (int)pieces(a.piece);
  a.give = kMostGiven / a.pieces;
  // The last launch: CTAs of a row, sixteen where that gives each two thousand columns, and one on an SM. Few rows come
  // to it as a rule, and their time is the call's: 85 us for 64 rows of which three do; 96 with clusters of 8, and
  // with two CTAs on an SM 97; one row that does 45, 55 and 49. Where all do, those leave less waiting: 16 rows 113,
  // 100 and 102 us, 64 rows 344, 248 and 280.
  int cluster = 1;
  while (vocab > (int64_t)cluster * kMaxShare || (cluster < kMaxCluster && vocab > cluster * 2048)) cluster *= 2;
  a.share = (int)((vocab + cluster - 1) / cluster + 3) / 4 * 4;
  a.run = (a.share + 4 * kThreads - 1) / (4 * kThreads) * 128;
  // what the launches tell one another: made by the context's first call and kept, so that a recorded
  // graph's addresses stay good
  constexpr size_t kBytes = (size_t)kRows * (kMaxPieces * 20 + kMostGiven * 8 + 24) + 16;
  if (!ctx->sample_ws) {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // (also while a stream is being recorded)
    GQ_CUDA_TRY(ctx, cudaThreadExchangeStreamCaptureMode(&mode));
    const cudaError_t e = cudaMalloc(&ctx->sample_ws, kBytes);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
      ctx->sample_ws = nullptr;
      return gq_cuda_fail(ctx, e, "sample_requests: cudaMalloc");
    }
  }
  a.piece_keys = static_cast<uint64_t *>(ctx->sample_ws);
  a.piece_mass = a.piece_keys + (size_t)kRows * kMostGiven;
  a.drawn = reinterpret_cast<double *>(a.piece_mass + (size_t)kRows * kMaxPieces);
  a.row_mass = reinterpret_cast<uint64_t *>(a.drawn + kRows);
  a.piece_top = reinterpret_cast<float *>(a.row_mass + kRows);
  a.piece_from = a.piece_top + (size_t)kRows * kMaxPieces;
  a.piece_given = reinterpret_cast<int32_t *>(a.piece_from + (size_t)kRows * kMaxPieces);
  a.todo = a.piece_given + (size_t)kRows * kMaxPieces;
  a.n_todo = a.todo + kRows;
  static bool attr_set[64] = {};
  if (!attr_set[ctx->device & 63]) {
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(finish_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostGiven * 16));
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_requests_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)));
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_requests_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    attr_set[ctx->device & 63] = true;
  }
  for (int64_t r0 = 0; r0 < m; r0 += kRows) {
    const int64_t rows = std::min<int64_t>(m - r0, kRows);
    Args b = a;
    b.logits += r0 * ld;
    if (b.temperature) b.temperature += r0;
    if (b.top_k) b.top_k += r0;
    if (b.top_p) b.top_p += r0;
    if (b.min_p) b.min_p += r0;
    if (b.uniforms) b.uniforms += r0;
    if (b.rng) b.rng += r0;
    b.tokens += r0;
    if (b.probs) b.probs += r0;
    GQ_CUDA_TRY(ctx, gq_launch(ctx, survey_kernel, dim3((unsigned)(rows * a.pieces)), dim3(kSurvey), (size_t)a.piece * 4, b));
    GQ_CUDA_TRY(ctx, gq_launch(ctx, finish_kernel, dim3((unsigned)rows), dim3(kThreads), (size_t)kMostGiven * 16, b));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(rows, std::max(1, ctx->num_sms / cluster)) * cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 2 : 1;
    GQ_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, sample_requests_kernel, (const Args)b));
  }
  return GQ_OK;
}
