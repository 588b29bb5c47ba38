// Rows of logits under temperature, top-k, top-p and min-p on gfx950: tokens drawn from given uniform numbers, the
// distribution they are drawn from, or the row with what the rules leave out at -inf.
//
// Mathematics. w_i = exp((l_i - max l) / T). The order: logits descending, the lower index first among equals. Every rule
// keeps a beginning of it: top-k its first k tokens, min-p those with w >= min_p, top-p, of what these two leave, with mass
// Z1, the tokens with less than top_p Z1 before them. The first token is always kept. So a row's outcome is one place of the
// order, the cut (a logit and, among its equals, an index), and the mass Z up to it. A draw is the first token of the
// order whose running mass exceeds coin Z. T not above 0, or a maximum that is not finite: the argmax alone.
//
// Masses are whole numbers, w in units of 2^-45 rounded once from 64 bits: their sums are exact, the same in any order
// and by any path below, and a row of 2^18 tokens stays under 2^64. What a token's rounding (2^-46 of the row's largest
// mass) can move is a comparison whose two sides are that close.
//
// A workgroup takes a row and passes over it as seldom as its rules allow, loads always in flight; nothing but the outcome goes
// to memory, and no workspace is needed:
//
// 1. One pass for the maximum, and each thread's own.
// 2. Where top-k (up to 768) or min-p leave few tokens, they bound the kept part by a logit before any weight is computed: the
//    k-th largest of the threads' maxima is not above the row's k-th logit, and min_p is a logit. A pass gathers what
//    lies above the bound into LDS (up to 2048 tokens), where it is sorted and everything is decided.
// 3. Otherwise a pass sums the row into bins, ordered by falling logit: 64 of them a factor of two in w, or, of bf16 rows of
//    magnitudes below 1024, one for each value, which are counted in 32 bits and weighed once each; where no rule bounds a
//    bf16 row, it is counted in pass 1, on the guess that its magnitudes are below 64. A place of the order is found in its bin:
//    by arithmetic, and a count of equals by index, where the bin is one value; gathered and sorted where it holds few tokens;
//    divided into 2048 ranges of logits again where it holds many. Top-p alone takes its list from the bins and decides as in 2.
// 4. An output is filled and the listed tokens put in, or written in a last pass where no list holds all that is kept.
//
// What bounds it: 256 rows of 151936 bf16 logits, a draw and fp32 shares each (the least traffic: 233 MB, 46 us) take 58 us
// where top-k 20 keeps a list in every row, 70 with top-p 0.95 alone, 86 where all is kept; 1024 rows cut (94 us) 118 to 129 us: the
// second pass and the bins' LDS additions, beside HBM. A single row that top-k, min-p or T bounds takes 9 to 22 us: its passes' latency
// on one CU. One that no rule bounds takes 34 to 41 us in bf16, 53 to 90 in fp16 and 61 to 83 in fp32, which have no bins by value:
// all of it is counted or weighed by one CU, where more could share it with launches or a wait between them (not tried).
// Few rows with an output are shared by workgroups that all find the cut: 16 rows cut take 22 us.

#include <type_traits>

#include "vocab_row.h"

namespace {

using namespace e4vocab;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));

constexpr int NT = 1024, kWaves = NT / 64;
constexpr int kBins = 4096, kList = 2048;
constexpr double kUnit = 0x1p45;
constexpr uint32_t kLowestKey = 0x007fffffu;  // of -inf

// A value that all threads have alike, in scalar registers.
template <typename U>
E4_DEV U uniform(U x) {
  static_assert(sizeof(U) == 4 || sizeof(U) == 8, "one word or two");
  if constexpr (sizeof(U) == 4) {
    return __builtin_bit_cast(U, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
  } else {
    const uint64_t w = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(w)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(w >> 32));
    return __builtin_bit_cast(U, static_cast<uint64_t>(hi) << 32 | lo);
  }
}

// A logit as a whole number of the same order; NaN the largest, both zeros alike.
E4_DEV uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
E4_DEV float value_of(uint32_t key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu)); }

// A token's mass in units of 2^-45, and -64 log2 w as a whole number. With 64 log2 w = r - (64 q + j), |r| <= 1/2, the mass is roots[j] =
// 2^(-j/64), times 2^(r/64) by its series (the next term is below 10^-16), times 2^-q.
struct Weighed {
  int steps;  // -64 log2 w, rounded
  uint64_t mass;
};
E4_DEV Weighed weigh(float x, float top, double c, const double* roots) {
  double y = (static_cast<double>(x) - static_cast<double>(top)) * (c * 64.0);
  y = __builtin_fmax(y, -70400.0);  // (and for the NaN of -inf times a scale of 0)
  const double n = __builtin_rint(y), r = y - n;
  constexpr double k = 0.6931471805599453 / 64;
  double p = k * k * k * k * k / 120;
  p = __builtin_fma(p, r, k * k * k * k / 24);
  p = __builtin_fma(p, r, k * k * k / 6);
  p = __builtin_fma(p, r, k * k / 2);
  p = __builtin_fma(p, r, k);
  p = __builtin_fma(p, r, 1.0);
  const int steps = -static_cast<int>(n);
  p = __builtin_ldexp(p * roots[steps & 63], 45 - (steps >> 6)) + 0x1p52;  // rounds to a whole number in the low 52 bits
  return Weighed{steps, __builtin_bit_cast(uint64_t, p) & 0xfffffffffffffull};
}

// Bins of a row's logits, their numbers rising as the logits fall. By weight: 64 a factor of two. By value (bf16): a bin for every
// value of magnitude from 2^(high - 15) to below 2^high, one for the smaller ones and one for what lies below -2^high, which
// weighs nothing. There a row is counted, and every value weighed once.
struct Bins {
  static constexpr float kFirst = 64.f;
  static constexpr uint32_t kFirst16 = (127 + 6) << 7;
  static constexpr int kOctaves = 15, kValues = kOctaves * 128, kSmall = kValues, kRest = 2 * kValues + 1;  // bins of values: 0 .. kRest - 1
  bool by_value;
  float top;
  double c;
  uint32_t low16, high16;  // bf16 patterns of 2^(high - 15) and 2^high

  // Bins of a row that is counted before its maximum is known: of magnitudes below 64.
  E4_DEV Bins() : by_value(true), top(0.f), c(0.0), low16(kFirst16 - kValues), high16(kFirst16) {}
  // (`first`: those)
  E4_DEV Bins(bool values, float top_, float temperature, double c_, bool first) : by_value(false), top(top_), c(c_), low16(0), high16(0) {
    if (!values) return;
    // magnitudes up to 2^10 leave few of a row's logits among the small
    const float reach = reach_of(top, temperature);
    if (!(reach < 1024.f)) return;
    by_value = true;
    high16 = ((__float_as_uint(reach) >> 23) + 1) << 7;
    high16 = uniform(high16);
    high16 = high16 > 64 * 128 ? high16 : 64 * 128;
    if (first) high16 = kFirst16;
    low16 = high16 - kValues;
  }
  // The magnitude that a row's masses end at: nothing below top - 32 T has one (e^-32 is 2^-46.2).
  static E4_DEV float reach_of(float top, float temperature) {
    return uniform(__builtin_fmaxf(__builtin_fabsf(top), __builtin_fabsf(top - 32.5f * temperature)));
  }
  // A bf16 pattern's magnitude as steps from the small ones: 0 for them, kValues + 1 from 2^high on. (Positive ones do not come there.)
  E4_DEV int steps(uint32_t w) const {
    const int m = w & 0x7fffu, lo = static_cast<int>(low16) - 1, hi = high16;
    return (m < lo ? lo : m < hi ? m : hi) - lo;
  }
  E4_DEV int of(float x) const {
    if (by_value) {
      const int up = steps(__float_as_uint(x) >> 16);
      return kSmall + (x < 0.f ? up : -up);
    }
    const double y = (static_cast<double>(x) - static_cast<double>(top)) * (c * 64.0);
    const int steps = -static_cast<int>(__builtin_rint(__builtin_fmax(y, -70400.0)));
    return steps < kBins - 1 ? steps : kBins - 1;
  }
  // Two patterns at once: their steps, and their bins' places in an array of words, in bytes.
  E4_DEV void places(uint32_t w, u16x2& up, u16x2& at) const {
    const uint16_t lo = static_cast<uint16_t>(low16 - 1), hi = static_cast<uint16_t>(high16);
    const u16x2 m = __builtin_bit_cast(u16x2, w & 0x7fff7fffu);
    up = __builtin_elementwise_min(__builtin_elementwise_max(m, u16x2{lo, lo}), u16x2{hi, hi}) - u16x2{lo, lo};
    const u16x2 sign = __builtin_bit_cast(u16x2, __builtin_bit_cast(i16x2, w) >> 15);  // all ones below 0
    at = ((up ^ ~sign) - ~sign + u16x2{kSmall, kSmall}) << 2;
  }
  // Counts a vector's logits (those before the row's maximum is known may be above the bins: they go to the first, and the row is
  // counted again). Bits of those among the small, whose masses are not those of one value.
  template <bool kAbove, typename Inside>
  E4_DEV uint32_t count(uint32_t* counts, int e0, const u32x4& w, Inside, int vocab) const {
    u16x2 least = {0xffff, 0xffff};  // steps; 0: among the small ones
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u16x2 up, at;
      places(w[i], up, at);
      if constexpr (kAbove) at = __builtin_bit_cast(u16x2, __builtin_elementwise_max(__builtin_bit_cast(i16x2, at), i16x2{0, 0}));
      least = __builtin_elementwise_min(least, up);
      const uint32_t both = __builtin_bit_cast(uint32_t, at);
      char* const c8 = reinterpret_cast<char*>(counts);
      if (Inside::value || static_cast<uint32_t>(e0 + 2 * i) < static_cast<uint32_t>(vocab))
        atomicAdd(reinterpret_cast<uint32_t*>(c8 + (both & 0xffffu)), 1u);
      if (Inside::value || static_cast<uint32_t>(e0 + 2 * i + 1) < static_cast<uint32_t>(vocab))
        atomicAdd(reinterpret_cast<uint32_t*>(c8 + (both >> 16)), 1u);
    }
    uint32_t hits = 0;
    if (least[0] == 0 || least[1] == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) hits |= ((w[i / 2] >> (16 * (i % 2))) & 0x7fffu) < low16 ? 1u << i : 0u;
    }
    return hits;
  }
  E4_DEV bool one_value(int b) const { return by_value && b != kSmall && b < kRest; }
  E4_DEV float value(int b) const {
    const uint32_t w = b < kSmall ? low16 + (kSmall - 1 - b) : 0x8000u | (low16 + (b - kSmall - 1));
    return __uint_as_float(w << 16);
  }
};

struct Shared {
  alignas(16) uint64_t mass[kBins];  // running sums over the bins
  alignas(16) uint32_t count[kBins];
  union {
    struct {
      uint64_t entry[kList];  // (~key << 32) | index: ascending is the order
      uint64_t run[kList];    // running masses
    } list;
    struct {
      alignas(16) uint64_t mass[kBins];
      alignas(16) uint32_t count[kBins];
    } sub;
    uint32_t maxima[NT];
  };
  double roots[64];
  u32x4 ends[2];
  uint64_t wave64[kWaves];
  uint32_t wave32[kWaves];
  uint32_t listed;
  int found;
  float thr;
  uint64_t sum;
};

E4_DEV bool in_row(int e, int vocab) { return static_cast<uint32_t>(e) < static_cast<uint32_t>(vocab); }

// Element j of a vector.
template <typename T>
E4_DEV float pick(const u32x4& w, int j) {
  constexpr bool kWide = sizeof(typename T::storage) == 4;
  const int k = kWide ? j : j / 2;
  const uint32_t one = k & 1 ? w[1] : w[0], two = k & 1 ? w[3] : w[2], word = k & 2 ? two : one;
  if constexpr (kWide)
    return __uint_as_float(word);
  else
    return T::to_f32(static_cast<uint16_t>(j & 1 ? word >> 16 : word));
}

// A row as a workgroup's threads pass over it: the vectors wholly inside it from memory, the elements before the first and
// behind the last of those (at most one vector at each end) out of LDS, where they are put once.
template <typename T>
struct Rows {
  // A thread's vectors on their way: what the registers hold (fp16's conversions take a vector's more).
  static constexpr int VEC = Row<T>::VEC, kAhead = T::code == EAGLE4_F16 ? 2 : 3, kAheadWeighed = 2;
  using S = typename T::storage;
  Row<T> row;
  int begin, end;  // whole vectors
  u32x4* ends;     // LDS, two
  float top;
  double c;
  int tid;

  E4_DEV Rows(const void* logits, int64_t n, int64_t stride, int vocab, u32x4* lds, int tid_)
      : row(logits, n, stride, vocab), ends(lds), top(0.f), c(0.0), tid(tid_) {
    begin = row.past > 0 ? 1 : 0;
    end = (vocab + row.past) / VEC;
    if (tid < 2 * VEC) {
      const int e = end_first(tid / VEC) + tid % VEC;
      reinterpret_cast<S*>(ends)[tid] = in_row(e, vocab) ? row.p[e] : T::from_f32(-INFINITY);
    }
    __syncthreads();
  }
  static E4_DEV uint32_t lowest() {
    const float none = -INFINITY;
    if constexpr (VEC == 8)
      return T::pack(none, none);
    else
      return __float_as_uint(none);
  }
  // The first element of an end's vector; the row's size where there is none.
  E4_DEV int end_first(int side) const {
    if (side == 0) return row.past > 0 ? row.first(0) : row.vocab;
    return end >= begin && end < row.vectors ? row.first(end) : row.vocab;
  }

  // This thread's vector of chunk c: NT vectors from `begin` on, all of them in the row.
  E4_DEV u32x4 load(int c) const {  // (passes read a row again: temporal)
    return *reinterpret_cast<const u32x4*>(row.p + row.first(begin + tid) + static_cast<int64_t>(c) * (NT * VEC));
  }

  // f(first element, vector, whether it is known to be inside the row) for every vector, a thread's in ascending order but for the
  // row's two ends; -inf outside the row. Of `shares` workgroups the one with number `share` has every shares-th chunk. U
  // chunks are on their way all the time: each load takes the place of the one that is used up.
  template <int U, typename F>
  E4_DEV void each_vector(F&& f, int share = 0, int shares = 1) const {
    const int whole = end > begin ? (end - begin) / NT : 0;
    const int n = whole > share ? (whole - share + shares - 1) / shares : 0;  // chunks of this workgroup
    const int e0 = row.first(begin + tid);
    const auto chunk = [&](int j) { return share + shares * j; };
    const auto first = [&](int j) { return e0 + chunk(j) * (NT * VEC); };
    if (n > 0) {  // (past the last chunk: the last again, so that the loads on their way are U at every step)
      const auto ahead = [&](int j) { return load(chunk(j < n ? j : n - 1)); };
      u32x4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = ahead(u);
      for (int j = 0; j < n; j += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const u32x4 now = w[u];
          w[u] = ahead(j + U + u);
          if (j + u < n) f(first(j + u), now, std::true_type{});
        }
      }
    }
    // what is left: less than a chunk of whole vectors, and the ends
    if (whole % shares == share) {
      const int v = begin + whole * NT + tid;
      const uint32_t low = lowest();
      u32x4 last = {low, low, low, low};
      if (v < end) last = load(whole);
      f(v < end ? row.first(v) : row.vocab, last, std::false_type{});
    }
    if (tid < 2 && share == 0) f(end_first(tid), ends[tid], std::false_type{});
  }

  // f(first element, values)
  template <int U = kAhead, typename F>
  E4_DEV void each(F&& f, int share = 0, int shares = 1) const {
    each_vector<U>(
        [&](int e0, const u32x4& w, auto) {
          float x[VEC];
          Row<T>::widen(w, x);
          f(e0, x);
        },
        share, shares);
  }

  // f(element, value) for every element of a vector, a word at a time: what takes a weight of each element would not fit the
  // registers for a whole vector at once.
  template <typename Inside, typename F>
  E4_DEV void elements(int e0, u32x4 now, Inside, F&& f) const {
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      if constexpr (VEC == 4) {
        if (Inside::value || in_row(e0 + i, row.vocab)) f(e0 + i, __uint_as_float(now[0]));
      } else {
        const int e = e0 + 2 * i;
        if (Inside::value || in_row(e, row.vocab)) f(e, T::to_f32(static_cast<uint16_t>(now[0])));
        if (Inside::value || in_row(e + 1, row.vocab)) f(e + 1, T::to_f32(static_cast<uint16_t>(now[0] >> 16)));
      }
      now = u32x4{now[1], now[2], now[3], now[0]};
    }
  }
  template <typename F>
  E4_DEV void each_element(F&& f) const {
    each_vector<kAheadWeighed>([&](int e0, const u32x4& w, auto inside) { elements(e0, w, inside, f); });
  }

  // f(element, value) for the elements of a vector that `hits` has a bit for, few of them.
  template <typename F>
  E4_DEV void hit_elements(int e0, const u32x4& w, uint32_t hits, F&& f) const {
    while (hits != 0) {
      const int i = __builtin_ctz(hits);
      hits &= hits - 1;
      if (in_row(e0 + i, row.vocab)) f(e0 + i, pick<T>(w, i));
    }
  }
};

E4_DEV uint64_t shfl_up64(uint64_t x, int d) {
  const uint32_t lo = __shfl_up(static_cast<uint32_t>(x), d, 64), hi = __shfl_up(static_cast<uint32_t>(x >> 32), d, 64);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
template <typename U>
E4_DEV U wave_scan(U x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    U o;
    if constexpr (sizeof(U) == 8)
      o = shfl_up64(x, d);
    else
      o = __shfl_up(x, d, 64);
    if (lane >= d) x += o;
  }
  return x;
}
// Inclusive running sum over the workgroup's threads; every thread calls it.
template <typename U>
E4_DEV U block_scan(U x, U* part, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  x = wave_scan(x, lane);
  __syncthreads();  // (part may still be read)
  if (lane == 63) part[wave] = x;
  __syncthreads();
  for (int i = 0; i < wave; ++i) x += part[i];
  return x;
}

E4_DEV void clear(uint64_t* mass, uint32_t* count, int tid) {
  constexpr u32x4 none = {0u, 0u, 0u, 0u};
  for (int i = tid; i < kBins / 2; i += NT) reinterpret_cast<u32x4*>(mass)[i] = none;
  for (int i = tid; i < kBins / 4; i += NT) reinterpret_cast<u32x4*>(count)[i] = none;
}

// The bins' counts and masses become running sums.
E4_DEV void scan_bins(uint64_t* mass, uint32_t* count, Shared& s, int tid) {
  constexpr int P = kBins / NT;
  static_assert(P == 4, "a 16-byte piece of counts a thread");
  const int lane = tid & 63, wave = tid >> 6;
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  u64x2* const m = reinterpret_cast<u64x2*>(mass) + 2 * tid;
  u32x4* const k = reinterpret_cast<u32x4*>(count) + tid;
  u64x2 a = m[0], b = m[1];
  u32x4 c = *k;
  a[1] += a[0];
  b[0] += a[1];
  b[1] += b[0];
  c[1] += c[0];
  c[2] += c[1];
  c[3] += c[2];
  uint64_t mb = wave_scan(b[1], lane);
  uint32_t kb = wave_scan(c[3], lane);
  __syncthreads();
  if (lane == 63) {
    s.wave64[wave] = mb;
    s.wave32[wave] = kb;
  }
  __syncthreads();
  mb -= b[1];
  kb -= c[3];
  for (int i = 0; i < wave; ++i) {
    mb += s.wave64[i];
    kb += s.wave32[i];
  }
  m[0] = u64x2{a[0] + mb, a[1] + mb};
  m[1] = u64x2{b[0] + mb, b[1] + mb};
  *k = u32x4{c[0] + kb, c[1] + kb, c[2] + kb, c[3] + kb};
  __syncthreads();
}

// The first bin whose running mass, or count, exceeds `target` (the last bin where none does).
E4_DEV int find_bin(const uint64_t* mass, const uint32_t* count, bool by_mass, uint64_t target, Shared& s, int tid) {
  constexpr int P = kBins / NT;
  if (tid == 0) s.found = kBins - 1;
  __syncthreads();
  uint64_t before = 0;
  if (tid > 0) before = by_mass ? mass[P * tid - 1] : count[P * tid - 1];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const uint64_t run = by_mass ? mass[P * tid + i] : count[P * tid + i];
    if (run > target && (P * tid + i == 0 || before <= target)) s.found = P * tid + i;
    before = run;
  }
  __syncthreads();
  const int b = uniform(s.found);
  __syncthreads();
  return b;
}

// The lowest key in [lo, hi] for which `ok` holds, given that it holds for hi and for every key above one that it
// holds for. By one wave: 64 probes a round.
template <typename F>
E4_DEV uint32_t lowest_key(uint32_t lo, uint32_t hi, F&& ok) {
  const int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  while (lo < hi) {
    const uint64_t span = static_cast<uint64_t>(hi) - lo;
    const uint32_t at = lo + static_cast<uint32_t>(span * lane / 64);  // lane 0: lo; below hi
    const uint64_t good = __ballot(ok(at));
    if (good & 1) return uniform(lo);
    const int first = good == 0 ? 64 : __builtin_ctzll(good);
    hi = first == 64 ? hi : lo + static_cast<uint32_t>(span * first / 64);
    lo = lo + static_cast<uint32_t>(span * (first - 1) / 64) + 1;
  }
  return uniform(hi);
}

// The same, where `guess` is a logit near that key: one round of probes if it is within 32 keys.
template <typename F>
E4_DEV uint32_t lowest_key_near(float guess, uint32_t hi, F&& ok) {
  const uint32_t at = guess > -INFINITY ? key_of(guess) : 0u;  // (NaN: no guess)
  if (at > kLowestKey + 32 && at < hi - 32) {
    const int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    const uint64_t good = __ballot(ok(at - 32 + lane));
    if (good != 0 && !(good & 1)) return uniform(at - 32 + __builtin_ctzll(good));
  }
  return lowest_key(kLowestKey, hi, ok);
}

// The lowest key of the bins up to b, given the row's largest.
E4_DEV uint32_t lowest_of(const Bins& bins, int b, uint32_t top) {
  if (!bins.by_value) {
    if (b == kBins - 1) return kLowestKey;
    const float guess = static_cast<float>(static_cast<double>(bins.top) - (b + 0.5) / (bins.c * 64.0));
    return lowest_key_near(guess, top, [&](uint32_t k) { return bins.of(value_of(k)) <= b; });
  }
  if (b >= Bins::kRest) return kLowestKey;
  return b == Bins::kSmall ? key_of(bins.value(b + 1)) + 1 : key_of(bins.value(b));
}

// The value of lane ^ J, by lane patterns: within a quad, a mirrored half row and quad, a row turned by 8, swaps of rows.
template <int J>
E4_DEV uint32_t partner32(uint32_t x, int lane) {
  const int v = static_cast<int>(x);
  if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);
  if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);
  if constexpr (J == 4) return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true), 0x1B, 0xF, 0xF, true);
  if constexpr (J == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, true);
  if constexpr (J == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return lane & 16 ? r[0] : r[1];
  }
  if constexpr (J == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
template <int J>
E4_DEV uint64_t ordered(uint64_t x, bool up, int lane) {  // the lower of x and lane ^ J's where `up` and bit J agree
  const uint64_t o = static_cast<uint64_t>(partner32<J>(static_cast<uint32_t>(x >> 32), lane)) << 32 | partner32<J>(static_cast<uint32_t>(x), lane);
  const bool low = ((lane & J) == 0) == up;
  return low == (o < x) ? o : x;
}
// The steps of a merge within a wave, from lane distance J down.
template <int J>
E4_DEV uint64_t merge_wave(uint64_t x, bool up, int lane) {
  x = ordered<J>(x, up, lane);
  if constexpr (J > 1) x = merge_wave<J / 2>(x, up, lane);
  return x;
}
E4_DEV uint64_t sort_wave(uint64_t x, bool up, int lane) {
  x = merge_wave<1>(x, (lane & 2) == 0, lane);
  x = merge_wave<2>(x, (lane & 4) == 0, lane);
  x = merge_wave<4>(x, (lane & 8) == 0, lane);
  x = merge_wave<8>(x, (lane & 16) == 0, lane);
  x = merge_wave<16>(x, (lane & 32) == 0, lane);
  return merge_wave<32>(x, up, lane);
}

// Sorts s.list.entry[0 .. n) ascending; n at most kList. Every thread calls it. A bitonic network over the next power of two: an entry
// a thread (two beyond NT), steps within a wave by lane patterns, those between waves through LDS. (Every step through LDS behind a
// barrier: 256 entries 16 us.)
template <int E>
E4_DEV void sort_entries(Shared& s, int n, int size, int tid) {
  const int lane = tid & 63;
  uint64_t x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int at = tid + NT * e;
    x[e] = at < n ? s.list.entry[at] : ~0ull;
    if (at < size) x[e] = sort_wave(x[e], (at & 64) == 0, lane);
  }
  for (int k = 128; k <= size; k <<= 1) {
    for (int j = k >> 1; j >= 64; j >>= 1) {
      if (E == 2 && j == NT) {  // the thread's own two (the last merge: ascending)
        const uint64_t lo = x[0] < x[E - 1] ? x[0] : x[E - 1];
        x[E - 1] = x[0] < x[E - 1] ? x[E - 1] : x[0];
        x[0] = lo;
        continue;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) s.list.entry[tid + NT * e] = x[e];
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int at = tid + NT * e;
        const uint64_t o = s.list.entry[at ^ j];
        const bool low = ((at & j) == 0) == ((at & k) == 0);
        x[e] = low == (o < x[e]) ? o : x[e];
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (tid + NT * e < size) x[e] = merge_wave<32>(x[e], ((tid + NT * e) & k) == 0, lane);
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) s.list.entry[tid + NT * e] = x[e];
  __syncthreads();
}
E4_DEV void sort_list(Shared& s, int n, int tid) {
  int size = 64;
  while (size < n) size <<= 1;
  if (size <= NT)
    sort_entries<1>(s, n, size, tid);
  else
    sort_entries<2>(s, n, size, tid);
}

E4_DEV uint32_t entry_key(uint64_t e) { return ~static_cast<uint32_t>(e >> 32); }

// Gathers the elements with lo <= value <= hi, sorts them and leaves their running masses from `base` on. How many there
// are (past kList: nothing is listed).
template <typename T>
E4_DEV int list_range(const Rows<T>& r, Shared& s, float lo, float hi, uint64_t base) {
  const int tid = r.tid;
  __syncthreads();
  if (tid == 0) s.listed = 0;
  __syncthreads();
  const bool from_top = hi >= r.top;
  r.template each_vector<Rows<T>::kAhead>([&](int e0, const u32x4& w, auto) {
    constexpr int VEC = Row<T>::VEC;
    float x[VEC];
    Row<T>::widen(w, x);
    bool any;
    if (from_top) {
      float most = x[0];
#pragma unroll
      for (int i = 1; i < VEC; ++i) most = __builtin_elementwise_maximum(most, x[i]);
      any = most >= lo;
    } else {
      any = false;
#pragma unroll
      for (int i = 0; i < VEC; ++i) any |= x[i] >= lo && x[i] <= hi;
    }
    if (any) {
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) hits |= x[i] >= lo && x[i] <= hi ? 1u << i : 0u;
      r.hit_elements(e0, w, hits, [&](int e, float y) {
        const uint32_t at = atomicAdd(&s.listed, 1u);
        if (at < kList) s.list.entry[at] = (static_cast<uint64_t>(~key_of(y)) << 32) | static_cast<uint32_t>(e);
      });
    }
  });
  __syncthreads();
  const int n = uniform(s.listed);
  if (n > kList) return n;
  sort_list(s, n, tid);
  constexpr int P = kList / NT;
  uint64_t m[P], sum = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int at = P * tid + i;
    sum += at < n ? weigh(value_of(entry_key(s.list.entry[at])), r.top, r.c, s.roots).mass : 0;
    m[i] = sum;
  }
  const uint64_t before = block_scan(sum, s.wave64, tid) - sum + base;
#pragma unroll
  for (int i = 0; i < P; ++i) s.list.run[P * tid + i] = before + m[i];
  __syncthreads();
  return n;
}

// The first of the list's n entries whose running mass exceeds `target`; n - 1 where none does.
E4_DEV int list_find(const Shared& s, int n, uint64_t target) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s.list.run[mid] > target)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

struct Place {
  float x;
  int index;
  uint64_t run;  // mass up to it, its own with it
};

// The element of the row that is `rank`-th (from 0) by index among those equal to x: a pass counts them by parts of 256 elements, and
// a wave looks through the part.
constexpr int kPartBits = 8;
static_assert(EAGLE4_ROWS_MAX_VOCAB <= NT << kPartBits, "a part a thread");
template <typename T>
E4_DEV int nth_equal(const Rows<T>& r, Shared& s, float x, uint32_t rank) {
  constexpr int VEC = Row<T>::VEC;
  const int tid = r.tid;
  uint32_t* const part = s.sub.count;
  __syncthreads();
  part[tid] = 0;
  if (tid == 0) s.found = 0;
  __syncthreads();
  r.template each_vector<Rows<T>::kAhead>([&](int e0, const u32x4& w, auto inside) {
    float y[VEC];
    Row<T>::widen(w, y);
    uint32_t hits = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) hits |= y[i] == x ? 1u << i : 0u;
    if (hits == 0) return;
    if (decltype(inside)::value && e0 >> kPartBits == (e0 + VEC - 1) >> kPartBits)
      atomicAdd(&part[e0 >> kPartBits], static_cast<uint32_t>(__popc(hits)));
    else
      r.hit_elements(e0, w, hits, [&](int e, float) { atomicAdd(&part[e >> kPartBits], 1u); });
  });
  __syncthreads();
  const uint32_t own = part[tid], run = block_scan(own, s.wave32, tid);
  if (run > rank && run - own <= rank) {
    s.found = tid;
    s.listed = rank - (run - own);
  }
  __syncthreads();
  const int e1 = uniform(s.found) << kPartBits;
  uint32_t left = uniform(s.listed);
  __syncthreads();
  if (tid < 64) {
#pragma unroll
    for (int i = 0; i < (1 << kPartBits) / 64; ++i) {
      const int e = e1 + 64 * i + tid;
      const bool hit = in_row(e, r.row.vocab) && T::to_f32(r.row.p[e]) == x;
      const uint64_t all = __ballot(hit);
      const uint32_t before = __popcll(all & ((uint64_t{1} << tid) - 1));
      if (hit && before == left) s.found = e;
      left -= __popcll(all);  // (below 0, a large number: found already)
    }
  }
  __syncthreads();
  const int e = s.found;
  __syncthreads();
  return e;
}

// The first element of the order whose running mass (by_mass) or count exceeds `target`, which is below the row's. Without
// `index` the element's place among its equals may stay unknown (-1): a pass less.
template <typename T>
E4_DEV Place locate(const Rows<T>& r, const Bins& bins, Shared& s, bool by_mass, uint64_t target, bool index) {
  const int tid = r.tid;
  const int b = find_bin(s.mass, s.count, by_mass, target, s, tid);
  uint64_t mass = uniform(b > 0 ? s.mass[b - 1] : uint64_t{0});  // before the range
  uint32_t count = uniform(b > 0 ? s.count[b - 1] : 0u), inside = uniform(s.count[b]) - count;
  // the bin's keys; every wave finds them for itself
  const uint32_t top = key_of(r.top);
  uint32_t lo = kLowestKey, hi = top;
  if (bins.one_value(b)) {
    lo = hi = key_of(bins.value(b));
  } else {
    lo = lowest_of(bins, b, top);
    if (bins.of(r.top) < b) hi = lowest_of(bins, b - 1, top) - 1;
  }
  while (inside > kList && lo < hi) {
    const int shift = 32 - __builtin_clz(hi - lo) > 11 ? 32 - __builtin_clz(hi - lo) - 11 : 0;
    __syncthreads();
    clear(s.sub.mass, s.sub.count, tid);
    __syncthreads();
    r.each_element([&](int, float x) {
      const uint32_t k = key_of(x);
      if (k >= lo && k <= hi) {
        const uint32_t at = (hi - k) >> shift;
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.sub.mass[at]), weigh(x, r.top, r.c, s.roots).mass);
        atomicAdd(&s.sub.count[at], 1u);
      }
    });
    __syncthreads();
    scan_bins(s.sub.mass, s.sub.count, s, tid);
    const int at = find_bin(s.sub.mass, s.sub.count, by_mass, target - (by_mass ? mass : count), s, tid);
    const uint64_t m0 = uniform(at > 0 ? s.sub.mass[at - 1] : uint64_t{0});
    const uint32_t c0 = uniform(at > 0 ? s.sub.count[at - 1] : 0u);
    inside = uniform(s.sub.count[at]) - c0;
    mass += m0;
    count += c0;
    const uint32_t first = hi - (static_cast<uint32_t>(at) << shift);  // the range's highest key
    const uint32_t wide = (1u << shift) - 1;
    lo = first - lo < wide ? lo : first - wide;
    hi = first;
    __syncthreads();
  }
  Place p;
  if (lo == hi) {  // one logit, however often
    p.x = value_of(lo);
    const uint64_t each = weigh(p.x, r.top, r.c, s.roots).mass;
    uint64_t rank = by_mass ? (each > 0 ? (target - mass) / each : 0) : target - count;
    if (rank >= inside) rank = inside - 1;
    p.run = mass + (rank + 1) * each;
    p.index = -1;
    if (index) p.index = nth_equal(r, s, p.x, static_cast<uint32_t>(rank));
    return p;
  }
  // (-0's key belongs to no element, but -0 >= 0)
  const int n = list_range(r, s, value_of(lo), value_of(hi == 0x7fffffffu ? hi - 1 : hi), mass);
  int at = by_mass ? list_find(s, n, target) : static_cast<int>(static_cast<uint32_t>(target) - count);
  at = at < n ? at : n - 1;
  p.x = value_of(entry_key(s.list.entry[at]));
  p.index = static_cast<int>(static_cast<uint32_t>(s.list.entry[at]));
  p.run = s.list.run[at];
  __syncthreads();
  return p;
}

// The place of a draw's running mass: what exceeds coin Z (whole masses: what exceeds its whole part).
E4_DEV uint64_t target_of(float coin, uint64_t z) {
  const double t = static_cast<double>(coin) * static_cast<double>(z);
  if (!(t > 0.0)) return 0;
  const uint64_t u = t < 0x1p63 ? static_cast<uint64_t>(t) : z;
  return u < z ? u : z - 1;
}
// The mass that top-p asks for: the first token whose running mass exceeds this is the last one kept.
E4_DEV uint64_t nucleus_of(float p, uint64_t z) {
  const double t = __builtin_ceil(static_cast<double>(p) * static_cast<double>(z));
  if (!(t > 1.0)) return 0;
  const uint64_t u = t < 0x1p63 ? static_cast<uint64_t>(t) : z;
  return (u < z ? u : z) - 1;
}

// A logit that at least k of the row's reach, from the threads' own maxima: about the k-th largest of them. Of M threads' parts of
// a row some -M ln(1 - k / M) logits reach it, so beyond kMostByMaxima the list would not hold them.
constexpr int kMostByMaxima = 768;
E4_DEV float bound_of(Shared& s, float mine, int k, int tid) {
  s.maxima[tid] = key_of(mine);
  __syncthreads();
  if (tid < 64) {
    uint32_t x[kWaves];
#pragma unroll
    for (int i = 0; i < kWaves; ++i) x[i] = s.maxima[64 * i + tid];
    // at least k maxima reach lo: the least of them that is a number, where there are k; none passes hi
    uint32_t lo = 0xff7fffffu, hi = 0;
    int numbers = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      lo = x[i] > kLowestKey && x[i] < lo ? x[i] : lo;
      hi = x[i] > hi ? x[i] : hi;
      numbers += __popcll(__ballot(x[i] > kLowestKey));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t l = __shfl_xor(lo, d, 64), h = __shfl_xor(hi, d, 64);
      lo = l < lo ? l : lo;
      hi = h > hi ? h : hi;
    }
    lo = uniform(lo);
    hi = uniform(hi);
    if (numbers < k) lo = hi = kLowestKey;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      int n = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) n += __popcll(__ballot(x[i] >= mid));
      if (n >= k) {
        lo = mid;
        if (n <= k + k / 8 + 16) break;
      } else {
        hi = mid - 1;
      }
    }
    if (tid == 0) s.thr = value_of(lo);
  }
  __syncthreads();
  const float b = uniform(s.thr);
  __syncthreads();
  return b;
}

struct Cut {
  float x;  // kept: logits above it, and its equals up to the index
  int index;
  bool single;  // the index alone
};

// Writes N outputs: 16-byte stores (8 bytes of four 16-bit outputs) where all of them are inside and lie on such a boundary.
// Nontemporal where a wave's stores are whole lines.
template <typename U, int N>
E4_DEV void store_vector(U* out, int e0, int vocab, const U (&y)[N]) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  constexpr int kBytes = N * static_cast<int>(sizeof(U));
  static_assert(kBytes == 8 || kBytes % 16 == 0, "sizes of a vector of rows");
  U* const p = out + e0;
  if (e0 >= 0 && e0 + N <= vocab && reinterpret_cast<uintptr_t>(p) % (kBytes < 16 ? 8 : 16) == 0) {
    uint32_t w[kBytes / 4];
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) {
      if constexpr (sizeof(U) == 4)
        w[i] = __builtin_bit_cast(uint32_t, y[i]);
      else
        w[i] = static_cast<uint32_t>(y[2 * i]) | static_cast<uint32_t>(y[2 * i + 1]) << 16;
    }
    if constexpr (kBytes == 8) {
      __builtin_nontemporal_store(u32x2{w[0], w[1]}, reinterpret_cast<u32x2*>(p));
    } else if constexpr (kBytes == 16) {
      __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]}, reinterpret_cast<u32x4*>(p));
    } else {
#pragma unroll
      for (int k = 0; k < kBytes / 16; ++k) reinterpret_cast<u32x4*>(p)[k] = u32x4{w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in_row(e0 + i, vocab)) p[i] = y[i];
  }
}

// What is written in a token's place: its share of the mass, or its logit.
template <typename T, typename P_>
struct ProbOut {
  using P = P_;
  using S = typename P::storage;
  S* out;
  float top;
  double c, unit;
  bool single;
  static E4_DEV S none() { return P::from_f32(0.f); }
  E4_DEV S operator()(float x) const {
    return P::from_f32(single ? 1.f : share(x));
  }
  E4_DEV float share(float x) const { return static_cast<float>(weight_of(x, top, c) * unit); }
};
template <typename T>
struct LogitOut {
  using S = typename T::storage;
  S* out;
  static E4_DEV S none() { return T::from_f32(-INFINITY); }
  E4_DEV S operator()(float x) const { return T::from_f32(x); }
};

// Writes a row of which all that is kept is s.list.entry[0 .. kept) or, kept 0, the token at cut.index alone: nothing of it is read
// again. The row is filled, then the kept tokens are put in.
template <typename Out>
E4_DEV void write_few(const Shared& s, int kept, const Cut& cut, int vocab, const Out& out, int share, int shares, int tid) {
  using S = typename Out::S;
  constexpr int N = 16 / sizeof(S);
  const int past = static_cast<int>(reinterpret_cast<uintptr_t>(out.out) % 16 / sizeof(S)), vectors = (vocab + past + N - 1) / N;
  S y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = Out::none();
  for (int v = share * NT + tid; v < vectors; v += shares * NT) store_vector(out.out, v * N - past, vocab, y);
  // Every wave waits for its own fill to arrive, then for the others', so that no token is overwritten. (A fence that other XCDs
  // see writes the fill back from the cache: 70 us and more here.)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const auto put = [&](int e, float x) {
    if ((e + past) / N / NT % shares == share) out.out[e] = out(x);
  };
  if (kept == 0) {
    if (tid == 0) put(cut.index, cut.x);
  } else {
    for (int i = tid; i < kept; i += NT)
      put(static_cast<int>(static_cast<uint32_t>(s.list.entry[i])), value_of(entry_key(s.list.entry[i])));
  }
}

// Writes a row of which much is kept.
template <typename T, typename Out>
E4_DEV void write_row(const Rows<T>& r, const Cut& cut, const Out& out, int share, int shares) {
  constexpr int VEC = Row<T>::VEC;
  using S = typename Out::S;
  r.template each<Rows<T>::kAheadWeighed>([&](int e0, const float(&x)[VEC]) {
    float left[VEC];  // the kept logits, the others at -inf
    S y[VEC];
    bool any = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const bool kept = x[i] > cut.x || (x[i] == cut.x && e0 + i <= cut.index);
      any |= kept;
      left[i] = kept ? x[i] : -INFINITY;
      y[i] = Out::none();
    }
    if (any) {
#pragma unroll 1
      for (int j = 0; j < VEC; ++j) {  // one weight at a time, for the registers
        const S one = left[0] == -INFINITY ? Out::none() : out(left[0]);
#pragma unroll
        for (int i = 0; i + 1 < VEC; ++i) {
          left[i] = left[i + 1];
          y[i] = y[i + 1];
        }
        y[VEC - 1] = one;
      }
    }
    store_vector(out.out, e0, r.row.vocab, y);
  }, share, shares);
}

// The same of probabilities where the bins are bf16 values: every value's share is computed once, into the counts' place. (Rows that
// keep all of 151936 tokens, 256 of them, fp32 shares: 104 -> 93 us.)
template <typename T, typename Out>
E4_DEV void write_shares(const Rows<T>& r, const Cut& cut, Shared& s, const Bins& bins, const Out& out, int share, int shares) {
  constexpr int VEC = Row<T>::VEC;
  using S = typename Out::S;
  float* const table = reinterpret_cast<float*>(s.count);
  __syncthreads();
  for (int i = r.tid; i <= Bins::kRest; i += NT)
    table[i] = bins.one_value(i) ? out.share(bins.value(i)) : -1.f;  // below 0: of no one value, each for itself
  __syncthreads();
  r.template each_vector<Rows<T>::kAheadWeighed>([&](int e0, const u32x4& w, auto) {
    float p[VEC];
    bool other = false;
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      u16x2 up, at;
      bins.places(w[i / 2], up, at);
      const uint32_t both = __builtin_bit_cast(uint32_t, at);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float x = T::to_f32(static_cast<uint16_t>(w[i / 2] >> (16 * j)));
        const bool kept = x > cut.x || (x == cut.x && e0 + i + j <= cut.index);
        const float q = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(table) + (j ? both >> 16 : both & 0xffffu));
        p[i + j] = kept ? q : 0.f;
        other |= p[i + j] < 0.f;
      }
    }
    if (other) {
#pragma unroll 1
      for (int j = 0; j < VEC; ++j) {  // (one at a time, for the registers)
        const float q = p[0] < 0.f ? out.share(pick<T>(w, j)) : p[0];
#pragma unroll
        for (int i = 0; i + 1 < VEC; ++i) p[i] = p[i + 1];
        p[VEC - 1] = q;
      }
    }
    S y[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) y[i] = Out::P::from_f32(p[i]);
    store_vector(out.out, e0, r.row.vocab, y);
  }, share, shares);
}

template <typename T>
__global__ __launch_bounds__(NT) void sample_rows_kernel(const eagle4_sample_rows_args a, int shares) {
  __shared__ Shared s;
  constexpr int VEC = Row<T>::VEC;
  const int64_t n = blockIdx.x / static_cast<uint32_t>(shares);
  const int share = blockIdx.x % static_cast<uint32_t>(shares);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t entry = uniform(a.entries.ptr != nullptr ? e4::ld(a.entries, n) : n);
  if (entry < 0 || entry >= a.num_entries) {  // a padded row: tokens of 0, like any other for what looks them up next, and its logits
    if (a.tokens != nullptr && share == 0 && tid < a.draws) a.tokens[n * a.draws + tid] = 0;
    // (one by one, 768 such rows 244 us: whole vectors, as the other rows have them, cost those 0.3 us of 16 by their code alone)
    if (a.copy_padded != 0) {
      using S = typename T::storage;
      const S* const from = static_cast<const S*>(a.logits) + n * a.stride_row;
      S* const to = static_cast<S*>(a.out) + n * a.stride_out;
#pragma unroll 8
      for (int i = share * NT + tid; i < a.vocab; i += shares * NT) to[i] = from[i];
    }
    return;
  }
  const float temperature = uniform(a.temperature[entry]);
  const int k = uniform(a.top_k != nullptr ? a.top_k[entry] : 0);
  const float p = uniform(a.top_p != nullptr ? a.top_p[entry] : 1.f), m = uniform(a.min_p != nullptr ? a.min_p[entry] : 0.f);

  int64_t* const tokens = a.tokens != nullptr && share == 0 ? a.tokens + n * a.draws : nullptr;
  const float* const coins = a.coins != nullptr ? a.coins + n * a.draws : nullptr;
  if (tid < 64) s.roots[tid] = exp2(tid * -1.0 / 64);
  const float coin = tokens != nullptr && tid < a.draws ? coins[tid] : 0.f;  // (here, beside the row's first loads)
  Rows<T> r(a.logits, n, a.stride_row, a.vocab, s.ends, tid);
  const bool by_k = k > 0 && k < a.vocab, by_m = m > 0.f, by_p = p < 1.f;
  const bool asked = by_k || by_m || by_p || tokens != nullptr || a.out_kind == EAGLE4_ROWS_PROBS;
  bool bounded = by_m || (by_k && k <= kMostByMaxima);
  // bf16 rows that will need their bins are counted in the pass that finds the maximum: 256 rows drawn from whole 56 -> 48 us, by
  // top-p 0.95 48 -> 43 (rows with a bound wait for their rules before the first pass: one row's top-k 15.8 -> 16.1)
  bool counted = T::code == EAGLE4_BF16 && temperature > 0.f && asked && !bounded;
  float mine = -INFINITY;
  const auto most = [&](const float(&x)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) mine = __builtin_elementwise_maximum(mine, x[i]);
  };
  if (counted) {
    if constexpr (T::code == EAGLE4_BF16) {
      clear(s.mass, s.count, tid);
      if (tid == 0) s.listed = 0;
      __syncthreads();
      const Bins first;
      r.template each_vector<Rows<T>::kAhead>([&](int e0, const u32x4& w, auto inside) {
        float x[VEC];
        Row<T>::widen(w, x);
        most(x);
        r.hit_elements(e0, w, first.count<true>(s.count, e0, w, inside, a.vocab), [&](int, float x) {
          const uint32_t at = atomicAdd(&s.listed, 1u);
          if (at < kList) s.list.entry[at] = __float_as_uint(x);
        });
      });
    }
  } else {
    r.each([&](int, const float(&x)[VEC]) { most(x); });
  }
  {
    const float w = wave_max(mine);
    if (lane == 0) s.wave32[wave] = __float_as_uint(w);
    __syncthreads();
    float top = __uint_as_float(s.wave32[0]);
    for (int i = 1; i < kWaves; ++i) top = __builtin_elementwise_maximum(top, __uint_as_float(s.wave32[i]));
    r.top = uniform(top);
    r.c = uniform(scale_of(temperature));
    __syncthreads();
  }
  Cut cut{-INFINITY, INT32_MAX, false};
  int kept_list = 0;  // kept tokens, where all of them are in the list
  uint64_t z = static_cast<uint64_t>(kUnit);

  if (!(temperature > 0.f) || !(r.top < INFINITY) || r.top == -INFINITY) {  // the argmax alone
    if (tid == 0) s.found = INT32_MAX;
    __syncthreads();
    int at = INT32_MAX;
    r.template each_vector<Rows<T>::kAhead>([&](int e0, const u32x4& w, auto) {
      float x[VEC];
      Row<T>::widen(w, x);
      float most = x[0];
#pragma unroll
      for (int i = 1; i < VEC; ++i) most = __builtin_elementwise_maximum(most, x[i]);
      if (most == r.top || most != most) {
        uint32_t hits = 0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) hits |= (r.top != r.top ? x[i] != x[i] : x[i] == r.top) ? 1u << i : 0u;
        r.hit_elements(e0, w, hits, [&](int e, float) { at = e < at ? e : at; });
      }
    });
    if (at != INT32_MAX) atomicMin(&s.found, at);
    __syncthreads();
    cut.single = true;
    cut.index = s.found;
    cut.x = r.top;
    if (tokens != nullptr && tid < a.draws) tokens[tid] = cut.index;
  } else {
    // min-p: the lowest logit whose weight reaches it
    float lowest = -INFINITY;
    if (by_m) {
      const double want = m < 1.f ? static_cast<double>(m) : 1.0;
      lowest = uniform(value_of(lowest_key_near(r.top + logf(static_cast<float>(want)) * temperature, key_of(r.top),
                                                [&](uint32_t key) { return weight_of(value_of(key), r.top, r.c) >= want; })));
    }
    int listed = kList + 1;  // the list holds the order's beginning
    uint64_t z1 = 0;         // the mass that top-p is taken of, where it is known
    float bound = lowest;
    if (by_k && k <= kMostByMaxima) {
      const float b = bound_of(s, mine, k, tid);
      bound = uniform(b > bound ? b : bound);
    }
    const uint32_t small = counted ? uniform(s.listed) : 0;  // their values are in the list
    counted = counted && small <= kList && Bins::reach_of(r.top, temperature) < Bins::kFirst;
    const Bins bins(T::code == EAGLE4_BF16, r.top, temperature, r.c, counted);
    for (bool binned = !asked;;) {
      if (bounded) listed = list_range(r, s, bound, r.top, 0);
      if (listed <= kList || binned) break;
      if (!counted) {
        clear(s.mass, s.count, tid);
        __syncthreads();
      }
      if (bins.by_value) {
        const auto add_small = [&](float x) {
          atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[Bins::kSmall]), weigh(x, r.top, r.c, s.roots).mass);
        };
        if (counted) {
          for (uint32_t i = tid; i < small; i += NT) add_small(__uint_as_float(static_cast<uint32_t>(s.list.entry[i])));
        } else if constexpr (T::code == EAGLE4_BF16) {
          r.template each_vector<Rows<T>::kAhead>([&](int e0, const u32x4& w, auto inside) {
            r.hit_elements(e0, w, bins.count<false>(s.count, e0, w, inside, a.vocab), [&](int, float x) { add_small(x); });
          });
        }
        __syncthreads();
#pragma unroll 2
        for (int j = 0; j < kBins / NT; ++j) {  // (two together: a weight is a chain of 64-bit operations)
          const int i = tid + j * NT;
          const uint64_t mass = s.count[i] * weigh(bins.value(i), r.top, r.c, s.roots).mass;
          if (i != Bins::kSmall && i < Bins::kRest) s.mass[i] = mass;
        }
      } else {
        r.each_element([&](int, float x) {
          const Weighed w = weigh(x, r.top, r.c, s.roots);
          const int b = w.steps < kBins - 1 ? w.steps : kBins - 1;
          atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]), w.mass);
          atomicAdd(&s.count[b], 1u);
        });
      }
      __syncthreads();
      scan_bins(s.mass, s.count, s, tid);
      z1 = uniform(s.mass[kBins - 1]);
      binned = true;
      bounded = false;
      if (!by_k && !by_m && by_p) {  // the bins say where top-p's cut is at most
        const int b = find_bin(s.mass, s.count, true, nucleus_of(p, z1), s, tid);
        bounded = s.count[b] <= kList;
        if (bounded)
          bound = uniform(value_of(lowest_of(bins, b, key_of(r.top))));
      }
    }
    if (listed <= kList) {  // everything is decided in the list
      int kept = listed;
      if (by_k && k < kept) kept = k;
      if (by_m) {
        int lo = 0, hi = kept;  // the entries that min-p leaves
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (value_of(entry_key(s.list.entry[mid])) >= lowest)
            lo = mid + 1;
          else
            hi = mid;
        }
        kept = m > 1.f ? 1 : lo;
      }
      if (kept < 1) kept = 1;
      if (by_k || by_m) z1 = s.list.run[kept - 1];
      if (by_p) kept = list_find(s, kept, nucleus_of(p, z1)) + 1;
      z = s.list.run[kept - 1];
      kept_list = kept;
      const uint64_t last = s.list.entry[kept - 1];
      cut.x = value_of(entry_key(last));
      cut.index = static_cast<int>(static_cast<uint32_t>(last));
      if (tokens != nullptr && tid < a.draws) {
        const int at = list_find(s, kept, target_of(coin, z));
        tokens[tid] = static_cast<int64_t>(static_cast<uint32_t>(s.list.entry[at]));
      }
    } else if (asked) {  // one place after another: top-k's cut, min-p's, top-p's, the draws'
      int d = -3;
      while (d < 0 || (tokens != nullptr && d < a.draws)) {
        const int step = d++;
        bool by_mass = true;
        uint64_t target = 0;
        if (step == -3) {
          if (!by_k) continue;
          by_mass = false;
          target = static_cast<uint64_t>(k) - 1;
        } else if (step == -2) {
          if (!by_m || (cut.x >= lowest && m <= 1.f)) continue;
          if (m > 1.f) {  // the first token alone
            by_mass = false;
          } else {
            uint64_t sum = 0;
            r.each_element([&](int, float x) {
              if (x >= lowest) sum += weigh(x, r.top, r.c, s.roots).mass;
            });
            sum = block_scan(sum, s.wave64, tid);
            if (tid == NT - 1) s.sum = sum;
            __syncthreads();
            cut.x = lowest;
            cut.index = INT32_MAX;
            z1 = uniform(s.sum);
            __syncthreads();
            continue;
          }
        } else if (step == -1) {
          z = z1;
          if (!by_p) continue;
          target = nucleus_of(p, z1);
        } else {
          target = target_of(coins[step], z);
        }
        const Place at = locate(r, bins, s, by_mass, target, step >= 0 || a.out != nullptr);  // draws need no more of a cut than its mass
        if (step >= 0) {
          if (tid == 0) tokens[step] = at.index;
          continue;
        }
        cut.x = at.x;
        cut.index = at.index;
        z1 = z = at.run;
      }
    }
  }
  if (a.out == nullptr) return;
  const auto write_any = [&](const auto& out) {
    if (kept_list > 0 || cut.single)
      write_few(s, kept_list, cut, a.vocab, out, share, shares, tid);
    else
      write_row(r, cut, out, share, shares);
  };
  if (a.out_kind == EAGLE4_ROWS_LOGITS) {
    write_any(LogitOut<T>{static_cast<typename T::storage*>(a.out) + n * a.stride_out});
    return;
  }
  const double unit = kUnit / static_cast<double>(z);
  const Bins bins(T::code == EAGLE4_BF16, r.top, temperature, r.c, false);
  const auto write = [&](const auto& out) {
    if constexpr (T::code == EAGLE4_BF16)
      if (kept_list == 0 && !cut.single && bins.by_value) return write_shares(r, cut, s, bins, out, share, shares);
    write_any(out);
  };
  if (a.out_dtype == EAGLE4_F32)
    write(ProbOut<T, e4::F32>{static_cast<float*>(a.out) + n * a.stride_out, r.top, r.c, unit, cut.single});
  else if (a.out_dtype == EAGLE4_BF16)
    write(ProbOut<T, e4::Bf16>{static_cast<uint16_t*>(a.out) + n * a.stride_out, r.top, r.c, unit, cut.single});
  else
    write(ProbOut<T, e4::F16>{static_cast<uint16_t*>(a.out) + n * a.stride_out, r.top, r.c, unit, cut.single});
}

template <typename T>
int launch(const eagle4_sample_rows_args& a, hipStream_t s) {
  // Few rows with an output: several workgroups a row find the same cut, and each writes its part (not in place, where one
  // would write what another still reads). From 129 rows on, two workgroups a row would no longer run all at once.
  constexpr int kPart = NT * Row<T>::VEC;
  const int parts = (a.vocab + kPart - 1) / kPart;
  int shares = 1;
  if (a.out != nullptr && a.out != a.logits && a.rows <= 128) shares = static_cast<int>(256 / a.rows < parts ? 256 / a.rows : parts);
  sample_rows_kernel<T><<<static_cast<unsigned>(a.rows * shares), NT, 0, s>>>(a, shares);
  return E4_LAUNCH_STATUS();
}

}  // namespace

extern "C" int eagle4_sample_rows(const eagle4_sample_rows_args* a, void* stream) {
  if (a->rows == 0) return EAGLE4_OK;
  const auto lies = [](const void* p, int64_t stride, int dtype) {  // elements on their own size
    return reinterpret_cast<uintptr_t>(p) % (dtype == EAGLE4_F32 ? 4 : 2) == 0 && stride >= 0;
  };
  if (a->rows < 0 || a->rows > (1 << 20) || a->vocab < 1 || a->vocab > EAGLE4_ROWS_MAX_VOCAB || a->num_entries < 1 ||
      a->logits == nullptr || a->temperature == nullptr || !e4::is_float_dtype(a->dtype) ||
      !lies(a->logits, a->stride_row, a->dtype) || a->draws < 0 || a->draws > EAGLE4_ROWS_MAX_DRAWS ||
      (a->entries.ptr != nullptr && !e4::is_index_dtype(a->entries.dtype)) || (a->tokens == nullptr) != (a->draws == 0) ||
      (a->coins == nullptr) != (a->draws == 0) || (a->tokens == nullptr && a->out == nullptr))
    return EAGLE4_NOT_COVERED;
  if (a->out != nullptr &&
      ((a->out_kind != EAGLE4_ROWS_PROBS && a->out_kind != EAGLE4_ROWS_LOGITS) || !e4::is_float_dtype(a->out_dtype) ||
       (a->out_kind == EAGLE4_ROWS_LOGITS && a->out_dtype != a->dtype) || !lies(a->out, a->stride_out, a->out_dtype) ||
       (a->rows > 1 && a->stride_out < a->vocab)))
    return EAGLE4_NOT_COVERED;
  if (a->copy_padded != 0 && (a->out == nullptr || a->out_kind != EAGLE4_ROWS_LOGITS)) return EAGLE4_NOT_COVERED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case EAGLE4_BF16: return launch<e4::Bf16>(*a, s);
    case EAGLE4_F16: return launch<e4::F16>(*a, s);
    default: return launch<e4::F32>(*a, s);
  }
}
