// Verification of a drafted tree by sampling on gfx950: the walk of a request's tree that leaves every emitted token
// distributed as the target's own, from given uniform numbers.
//
// Mathematics. p = softmax(l / T) of a visited row. Its children are tried in row order against the residual r, first p, of
// mass Z, first 1: a child of token x and coin u is accepted iff u q(x) Z < r(x). q is what the children were drawn from:
//   - given draft probabilities: a rejection leaves r <- max(r - Z q, 0). With s the sum of the Z so far that is
//     max(p - s q, 0), so one number carries all rejections of a row;
//   - none given: the drafted token alone (q(x) = 1); a rejection leaves r(x) = 0.
// When no child is accepted, the walk ends with the first token t with r(0) + .. + r(t) > w Z, w the request's final coin.
// (Z = 0, which only rounding or a q that is no distribution leaves: p again.) T = 0, or a row whose maximum is not
// finite: all mass on the argmax (first index, NaN the largest), as greedy acceptance has it.
//
// Decisions are comparisons, so everything that enters them is held in 64 bits: exp2 is a polynomial there (16 operations
// an element at the rate of 32-bit ones, against about 10 with the hardware's 32-bit exp2, whose error would flip one
// comparison in 10^7, and of a flat row's running sums far more).
//
// Split: a wave takes 4096 elements of a row, a chunk. Three kinds of launches:
//   - statistics: of every chunk of a row its maximum and its mass relative to that. All rows of all trees at once, or the
//     trees' first rows and later those that may still be visited: the walk visits a few of them, but one after another,
//     and a workgroup that reads its request's rows on its own has one CU's rate (vocabulary 151936, bf16: one tree of
//     16 rows 105 to 232 us that way, by the walk's length, against 20; 64 trees of up to 16 rows 228 against 87);
//   - the walk, a workgroup per request: the rows' sums out of the chunks', then the decisions, a lane a child. Ends with the
//     final token: the chunks' running sum leads to one chunk, which is read. With draft probabilities a rejection needs the
//     residual's mass: the walk stops there and leaves its state;
//   - the residual's launch sums max(p - s q, 0) over the chunks of the stopped walks, and the walk is launched again.
// After kPairs such pairs a walk reads the rows of its further rejections itself. None, one and two pairs take 87, 62 and
// 65 us for 32 chains of 6 (one rejection each at most), 80, 78 and 76 for 12 trees of 12 over 50257 tokens, 200, 176 and 151
// for 16 trees of 16 over 151936. Continuing the walk in the residual's last workgroup instead of a launch of its own takes a
// fence of every workgroup, and those cost more (95 us instead of 71). The walk's workgroup has 512 threads for those rows:
// with 256, 89 us instead of 76 for the 12 trees; with 1024, 3% off the trees and 10% on single users' walks.
// What bounds it: the statistics by their 64-bit operations (87 us for 750 rows, 44 of them the logits' own; a table
// of 32 roots with a polynomial of degree 4 has a third fewer operations and is no faster for its lookups; one chunk
// loaded ahead of another, 93 us), the walk by its chain of dependent loads (13 us for one request, 21 among 64).

#include "vocab_row.h"

namespace {

using namespace e4vocab;

struct NoQ {  // no draft probabilities
  using storage = uint16_t;
  static constexpr int code = -1;
  static E4_DEV float to_f32(storage) { return 0.f; }
};

constexpr int kChunk = 4096;  // elements
constexpr int kPart = 1024;   // of a residual's masses
constexpr int kParts = kChunk / kPart;

// 64 NV vectors of a row from `v0` on: lane l has v0 + l, v0 + l + 64, ..; all loads are in flight together. -inf outside
// the row.
template <typename T, int NV>
E4_DEV void load_vectors(const Row<T>& row, int v0, int lane, u32x4 (&w)[NV]) {
  if (row.first(v0) >= 0 && row.first(v0 + 64 * NV) <= row.vocab) {  // wholly inside
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = row.raw(v0 + lane + 64 * i);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = row.load(v0 + lane + 64 * i);
  }
}

// The draft's probabilities of the same elements; `wide` where their vectors lie on vector boundaries too (rows of one
// stride over bases on 16 bytes do).
template <typename Q, int VEC>
struct QRow {
  using S = typename Q::storage;
  const S* p;
  bool wide;
  E4_DEV QRow(const void* probs, int64_t row, int64_t stride, int past) {
    p = static_cast<const S*>(probs) + row * stride;
    constexpr uintptr_t kTo = VEC * sizeof(S) < 16 ? VEC * sizeof(S) : 16;
    wide = reinterpret_cast<uintptr_t>(p - past) % kTo == 0;
  }
  E4_DEV void load(int e0, int vocab, float (&q)[VEC]) const {
    if (wide && e0 >= 0 && e0 + VEC <= vocab) {
      constexpr int kWords = VEC * static_cast<int>(sizeof(S)) / 4;
      uint32_t w[kWords];
      if constexpr (kWords == 2) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(p + e0);
        w[0] = v[0];
        w[1] = v[1];
      } else {
#pragma unroll
        for (int k = 0; k < kWords / 4; ++k) {
          const u32x4 v = reinterpret_cast<const u32x4*>(p + e0)[k];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[4 * k + i] = v[i];
        }
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if constexpr (sizeof(S) == 4)
          q[i] = __uint_as_float(w[i]);
        else
          q[i] = Q::to_f32(static_cast<S>(w[i / 2] >> (16 * (i % 2))));
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) q[i] = e0 + i >= 0 && e0 + i < vocab ? Q::to_f32(p[e0 + i]) : 0.f;
    }
  }
};

constexpr int kMaxRows = 64;  // of a tree: a lane each
constexpr int64_t kTwoSteps = 1 << 14;  // chunks of a launch
constexpr int kPairs = 2;     // residual and walk launches behind the first walk
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kWalkThreads = 512, kWalkWaves = kWalkThreads / 64;

// A stopped walk, `count` rows on its path. kForMass: the last one is `node`, whose child `child` was rejected last. kForRows:
// it goes on with `node`; `rows` has a bit for it and for each of its descendants.
constexpr int kForMass = 1, kForRows = 2;
struct State {
  int32_t stopped, node, child, count;
  double spent;
  uint64_t rows;
  float top;  // the row's maximum
};

struct Split {
  int chunks;  // of a row
  int64_t maxes_off, masses_off, state_off;  // in the workspace, bytes; the chunks' sums come first
};

struct Work {  // a row's parts of the workspace
  const double* sums;
  const float* maxes;
  E4_DEV Work(const eagle4_sample_tree_args& a, const Split& s, int64_t row) {
    sums = reinterpret_cast<const double*>(a.workspace) + row * s.chunks;
    maxes = reinterpret_cast<const float*>(static_cast<const char*>(a.workspace) + s.maxes_off) + row * s.chunks;
  }
};

// The request of a logits row: how many of them end at it or before. 64 probes at a time.
E4_DEV int request_of(const eagle4_sample_tree_args& a, int64_t row, int lane) {
  int lo = 0, n = a.num_reqs;  // it is lo .. lo + n, the last one: none
  while (n > 0) {
    const int step = (n + 63) / 64, at = lo + lane * step + step - 1;  // ends at row or before: lo is behind it
    const bool past = at < lo + n && e4::ld(a.cu_num_logits, at + 1) <= row;
    const int whole = __popcll(__ballot(past));
    lo += whole * step;
    n = n - whole * step < step - 1 ? n - whole * step : step - 1;
  }
  return lo;
}

E4_DEV int wave_min(int x) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const int o = __shfl_xor(x, k, 64);
    x = o < x ? o : x;
  }
  return x;
}

// Maximum and mass of a chunk of row n, by one wave, from its vectors as loaded. Where all mass is on one element (T = 0, a
// maximum of +inf or NaN) the place of the sum holds the first index of the maximum.
template <typename T, int NV>
E4_DEV void chunk_statistics(const eagle4_sample_tree_args& a, const Split& s, int64_t n, int chunk, const Row<T>& row,
                             const u32x4 (&w)[NV], float temperature, int lane) {
  constexpr int VEC = Row<T>::VEC;
  float x[NV][VEC];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    Row<T>::widen(w[i], x[i]);
#pragma unroll
    for (int k = 0; k < VEC; ++k) m = __builtin_elementwise_maximum(m, x[i][k]);
  }
  m = wave_max(m);
  double sum = 0.0;
  if (!(temperature > 0.f) || !(m < INFINITY)) {
    int at = INT32_MAX;
#pragma unroll
    for (int i = NV - 1; i >= 0; --i)
#pragma unroll
      for (int k = VEC - 1; k >= 0; --k) {
        const int e = row.first((chunk * NV + i) * 64 + lane) + k;
        if (e >= 0 && e < row.vocab && (m != m ? x[i][k] != x[i][k] : x[i][k] == m)) at = e;
      }
    sum = wave_min(at);
  } else {
    const double c = scale_of(temperature);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum += weight_of(x[i][k], m, c);
    sum = wave_sum(sum);
  }
  if (lane == 0) {
    const Work out(a, s, n);
    const_cast<double*>(out.sums)[chunk] = sum;
    const_cast<float*>(out.maxes)[chunk] = m;
  }
}

// Of every row that a walk can visit.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_chunks(const eagle4_sample_tree_args a, const Split s) {
  constexpr int NV = kChunk / Row<T>::VEC / 64;
  const int lane = threadIdx.x & 63;
  const uint32_t id = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n = id / static_cast<uint32_t>(s.chunks);
  const int chunk = static_cast<int>(id - n * s.chunks);
  if (n >= a.rows) return;
  const Row<T> row(a.logits, n, a.stride_row, a.vocab);
  u32x4 w[NV];
  load_vectors<T, NV>(row, chunk * (64 * NV), lane, w);
  const int b = __builtin_amdgcn_readfirstlane(request_of(a, n, lane));
  if (b >= a.num_reqs || n - e4::ld(a.cu_num_logits, b) >= a.width) return;  // a row that no walk visits
  chunk_statistics<T, NV>(a, s, n, chunk, row, w, a.temperature[b], lane);
}

// Of the trees' first rows (first != 0), or of the rows that the stopped walks may still visit.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_chunks_of(const eagle4_sample_tree_args a, const Split s, int first) {
  constexpr int NV = kChunk / Row<T>::VEC / 64;
  const int lane = threadIdx.x & 63, r = blockIdx.y, b = blockIdx.z;
  const int chunk = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (chunk >= s.chunks) return;
  if (!first) {
    const State* const st = reinterpret_cast<const State*>(static_cast<char*>(a.workspace) + s.state_off) + b;
    if (st->stopped != kForRows || !(st->rows >> r & 1)) return;
  }
  const int64_t start = e4::ld(a.cu_num_logits, b), end = e4::ld(a.cu_num_logits, b + 1), n = start + r;
  if (start < 0 || n >= end || end > a.rows) return;
  const Row<T> row(a.logits, n, a.stride_row, a.vocab);
  u32x4 w[NV];
  load_vectors<T, NV>(row, chunk * (64 * NV), lane, w);
  chunk_statistics<T, NV>(a, s, n, chunk, row, w, a.temperature[b], lane);
}

// The residual of a vector's elements out of its logits, times the row's total; `top` is the row's maximum.
template <typename Q, int VEC>
E4_DEV void residual(const float (&x)[VEC], const QRow<Q, VEC>& qrow, int first, int vocab, double c, float top, double spent,
                     double (&r)[VEC]) {
  if constexpr (Q::code >= 0) {
    float q[VEC];
    if (spent > 0.0) qrow.load(first, vocab, q);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      r[i] = weight_of(x[i], top, c);
      if (spent > 0.0) r[i] = __builtin_fmax(r[i] - spent * static_cast<double>(q[i]), 0.0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) r[i] = weight_of(x[i], top, c);
  }
}

E4_DEV double* masses_of(const eagle4_sample_tree_args& a, const Split& s, int b) {  // of request b's stopped row
  return reinterpret_cast<double*>(static_cast<char*>(a.workspace) + s.masses_off) + static_cast<int64_t>(b) * s.chunks * kParts;
}

// Those elements of a vector away that are the `token` of a lane of `gone`.
template <int VEC>
E4_DEV void take_out(float (&x)[VEC], int first, uint64_t gone, int token) {
  for (; gone != 0; gone &= gone - 1) {
    const int at = __builtin_amdgcn_readlane(token, __builtin_ctzll(gone)) - first;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i == at) x[i] = -INFINITY;
  }
}

// The mass of it in 64 NV vectors from v0 on, by one wave; their loads are in flight together. `gone`: the lanes whose `token`
// is taken out.
template <typename T, typename Q, int NV>
E4_DEV double residual_mass(const Row<T>& row, const QRow<Q, Row<T>::VEC>& qrow, int v0, double c, float top, double spent,
                            int lane, uint64_t gone, int token) {
  constexpr int VEC = Row<T>::VEC;
  u32x4 w[NV];
  load_vectors<T, NV>(row, v0, lane, w);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int first = row.first(v0 + lane + 64 * i);
    float x[VEC];
    Row<T>::widen(w[i], x);
    if constexpr (Q::code < 0) take_out<VEC>(x, first, gone, token);
    double r[VEC];
    residual<Q, VEC>(x, qrow, first, row.vocab, c, top, spent, r);
#pragma unroll
    for (int k = 0; k < VEC; ++k) sum += r[k];
  }
  return wave_sum(sum);
}

template <typename T, typename Q>
__global__ __launch_bounds__(kThreads) void sample_residual(const eagle4_sample_tree_args a, const Split s) {
  constexpr int VEC = Row<T>::VEC;
  const int lane = threadIdx.x & 63, b = blockIdx.y;
  const int part = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* const work = static_cast<char*>(a.workspace);
  const State st = reinterpret_cast<const State*>(work + s.state_off)[b];
  if (st.stopped != kForMass || part >= s.chunks * kParts) return;
  const int64_t n = e4::ld(a.cu_num_logits, b) + st.node;
  const Row<T> row(a.logits, n, a.stride_row, a.vocab);
  const QRow<Q, Row<T>::VEC> qrow(a.probs, n, a.stride_prob, row.past);
  const double c = scale_of(a.temperature[b]);
  const double mass = residual_mass<T, Q, kPart / VEC / 64>(row, qrow, part * (kPart / VEC), c, st.top, st.spent, lane, 0, 0);
  if (lane == 0) masses_of(a, s, b)[part] = mass;
}

// The walk. Every wave takes the decisions, lane j for row j of the tree; the waves part for the rows' sums and for the
// final token's chunk.
template <typename T, typename Q>
__global__ __launch_bounds__(kWalkThreads) void sample_walk(const eagle4_sample_tree_args a, const Split s, int first, int last, int roots) {
  constexpr int VEC = Row<T>::VEC, NV = (kChunk / VEC + kWalkThreads - 1) / kWalkThreads;  // vectors of a thread in the final token's chunk
  constexpr bool kProbs = Q::code >= 0;
  __shared__ float s_top[kMaxRows];
  __shared__ double s_total[kMaxRows];
  __shared__ int s_lost_chunk[kMaxRows];
  __shared__ double s_lost_mass[kMaxRows];
  __shared__ double s_scan[kWalkWaves];
  __shared__ int s_token, s_last;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* const work = static_cast<char*>(a.workspace);
  State* const state = reinterpret_cast<State*>(work + s.state_off) + b;
  double* const masses = masses_of(a, s, b);
  int node = 0, count = 0, resumed = 0;
  double spent = 0.0;
  uint64_t have = roots ? 1 : ~0ull;  // rows whose statistics are there
  if (!first) {
    const State st = *state;
    if (st.stopped == 0) return;
    node = st.node;
    count = st.count;
    resumed = st.child;
    spent = st.spent;
    if (st.stopped == kForRows) have = st.rows;
  }

  const int64_t slot = e4::ld(a.idx_mapping, b);
  const int64_t start = e4::ld(a.cu_num_logits, b);
  const int64_t rows = e4::ld(a.cu_num_logits, b + 1) - start;
  const bool valid = slot >= 0 && slot < a.slots && start >= 0 && rows > 0 && start + rows <= a.rows;
  const int limit = !valid ? 0 : static_cast<int>(rows < a.width ? rows : a.width);
  const float temperature = a.temperature[b];
  const bool greedy = !(temperature > 0.f);
  const double c = scale_of(temperature);

  // lane j: row j's parent, token, coin, and of its parent's row the token's logit and draft probability
  int parent = -1;
  int64_t token = -1;
  float coin = 0.f, logit = 0.f, drawn = 1.f;
  if (lane < limit) {
    parent = static_cast<int>(e4::ld(a.parents, slot, lane));
    token = e4::ld(a.drafted, start + lane);
    coin = a.coins[start + lane];
  }
  const bool child = lane > 0 && lane < limit && parent >= 0 && parent < limit && token >= 0 && token < a.vocab;
  if (child) {
    logit = T::to_f32(static_cast<const typename T::storage*>(a.logits)[(start + parent) * a.stride_row + token]);
    if constexpr (kProbs)
      drawn = Q::to_f32(static_cast<const typename Q::storage*>(a.probs)[(start + parent) * a.stride_prob + token]);
  }

  // The rows' maxima and totals out of the chunks', 16 lanes a row; a row with all mass on one element: its index.
  for (int r = tid / 16; r < limit; r += kWalkThreads / 16) {
    if (!(have >> r & 1)) continue;
    const Work w(a, s, start + r);
    const int l16 = lane & 15;
    float top = -INFINITY;  // the lane's chunks', then the row's
    double total = 0.0;
    for (int k0 = l16; k0 < s.chunks; k0 += 64) {
      float m[4], most = top;
      double sum[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = k0 + 16 * i < s.chunks;
        m[i] = in ? w.maxes[k0 + 16 * i] : -INFINITY;
        sum[i] = in ? w.sums[k0 + 16 * i] : 0.0;
        most = __builtin_elementwise_maximum(most, m[i]);
      }
      total *= weight_of(top, most, c);
#pragma unroll
      for (int i = 0; i < 4; ++i) total += sum[i] * weight_of(m[i], most, c);
      top = most;
    }
    const float mine = top;
    top = max16(top);
    if (greedy || !(__builtin_fabsf(top) < INFINITY)) {
      int at = INT32_MAX;  // its first chunk's; a row of -inf: 0
      for (int k = l16; k < s.chunks; k += 16)
        if (at == INT32_MAX && (top != top ? w.maxes[k] != w.maxes[k] : w.maxes[k] == top)) at = k;
#pragma unroll
      for (int k = 1; k < 16; k <<= 1) {
        const int o = __shfl_xor(at, k, 64);
        at = o < at ? o : at;
      }
      total = top == -INFINITY ? 0.0 : w.sums[at];
    } else {
      total *= weight_of(mine, top, c);
      total = sum16(total);
    }
    if (l16 == 0) {
      s_top[r] = top;
      s_total[r] = total;
    }
  }
  __syncthreads();
  // the parent's p of the token times the parent's total
  const double p = weight_of(logit, child ? s_top[parent] : 0.f, c);

  const auto lane_f64 = [](double x, int j) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(bits), j);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(bits >> 32), j);
    return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
  };
  const auto out_token = [&](int64_t x) {
    if (tid == 0) a.sampled[b * a.stride_sampled + count - 1] = x;
  };
  const auto sum_of_masses = [&] {
    double sum = 0.0;
    for (int k = lane; k < s.chunks * kParts; k += 64) sum += masses[k];
    return wave_sum(sum);
  };

  while (count < limit || resumed > 0) {
    const Row<T> row(a.logits, start + node, a.stride_row, a.vocab);
    const QRow<Q, VEC> qrow(a.probs, start + node, a.stride_prob, row.past);
    const Work w(a, s, start + node);
    const float top = s_top[node];
    const double total = s_total[node];
    const bool single = greedy || !(__builtin_fabsf(top) < INFINITY);
    double mass = total;   // Z, and above s, times the total
    uint64_t rejected = 0; // tokens taken out of the residual (no draft probabilities)
    uint64_t kids = __ballot(child && parent == node);
    if (resumed > 0) {
      kids &= resumed < 63 ? ~0ull << (resumed + 1) : 0ull;
      mass = sum_of_masses();
      resumed = 0;
    } else {
      if (tid == 0) a.path[slot * a.stride_path + count] = node;
      ++count;
      spent = 0.0;
    }

    // the children, in row order
    int next = -1;
    if (single) {
      const uint64_t fits = kids & __ballot(token == static_cast<int64_t>(total));
      if (fits != 0 && count < limit) next = __builtin_ctzll(fits);
      kids = 0;
    }
    while (kids != 0 && count < limit) {
      const int j = __builtin_ctzll(kids);
      kids &= kids - 1;
      double r = lane_f64(p, j), q = 1.0;
      if constexpr (kProbs) {
        q = static_cast<double>(__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, drawn), j)));
        if (spent > 0.0) r = __builtin_fmax(r - spent * q, 0.0);
      } else {
        const int x = __builtin_amdgcn_readlane(static_cast<int>(token), j);
        if ((__ballot(static_cast<int>(token) == x) & rejected) != 0) r = 0.0;
      }
      const float u = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, coin), j));
      if (static_cast<double>(u) * q * mass < r) {
        next = j;
        break;
      }
      if constexpr (kProbs) {
        spent += mass;
        if (!last) {
          if (tid == 0) *state = State{kForMass, node, j, count, spent, 0, top};
          return;
        }
        __syncthreads();  // the last masses have been read
        for (int k = wave; k < s.chunks * kParts; k += kWalkWaves) {
          const double m = residual_mass<T, Q, kPart / VEC / 64>(row, qrow, k * (kPart / VEC), c, top, spent, lane, 0, 0);
          if (lane == 0) masses[k] = m;
        }
        __syncthreads();
        mass = sum_of_masses();
      } else if (r > 0.0) {
        rejected |= 1ull << j;
        mass = __builtin_fmax(mass - r, 0.0);
      }
    }
    if (next >= 0) {
      out_token(__shfl(token, next, 64));
      node = next;
      if (!(have >> node & 1)) {
        uint64_t under = 1ull << node, before = 0;
        while (under != before) {
          before = under;
          under |= __ballot(lane > 0 && lane < limit && parent >= 0 && parent < limit && (before >> parent & 1));
        }
        if (tid == 0) *state = State{kForRows, node, 0, count, 0.0, under, 0.f};
        return;
      }
      continue;
    }

    // no child accepted: the token of the final coin
    int64_t found = static_cast<int64_t>(total);
    if (!single) {
      int lost = 0;
      if constexpr (!kProbs) {  // the chunks that lost a token, summed again
        uint64_t left = rejected;
        const int my_chunk = static_cast<int>((token + row.past) / kChunk);
        while (left != 0) {
          const int k = __builtin_amdgcn_readlane(my_chunk, __builtin_ctzll(left));
          left &= ~__ballot(my_chunk == k);
          if (lost % kWalkWaves == wave) {
            const double sum = residual_mass<T, Q, kChunk / VEC / 64>(row, qrow, k * (kChunk / VEC), c, top, 0.0, lane, rejected,
                                                                               static_cast<int>(token));
            if (lane == 0) {
              s_lost_chunk[lost] = k;
              s_lost_mass[lost] = sum;
            }
          }
          ++lost;
        }
        if (lost > 0) __syncthreads();
      }
      // a chunk's mass, or of a residual a part's
      const auto mass_of = [&](int k) {
        if (spent > 0.0) return masses[k];
        double m = w.sums[k] * weight_of(w.maxes[k], top, c);
        for (int i = 0; i < lost; ++i)
          if (s_lost_chunk[i] == k) m = s_lost_mass[i];
        return m;
      };
      if (lost > 0) {
        mass = 0.0;
        for (int k = lane; k < s.chunks; k += 64) mass += mass_of(k);
        mass = wave_sum(mass);
      }
      if (!(mass > 0.0)) {  // p again
        spent = 0.0;
        rejected = 0;
        lost = 0;
        mass = total;
      }
      const double target = static_cast<double>(a.final_coins[b]) * mass;
      const int units = spent > 0.0 ? s.chunks * kParts : s.chunks, unit = (spent > 0.0 ? kPart : kChunk) / VEC;
      double base = 0.0;
      int at = -1, full = 0;  // the unit in which the running sum passes the target, the last one that has mass
      for (int k0 = 0; k0 < units && at < 0; k0 += 64) {
        const double m = k0 + lane < units ? mass_of(k0 + lane) : 0.0;
        double run = m;
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
          const double o = __shfl_up(run, k, 64);
          if (lane >= k) run += o;
        }
        const uint64_t passed = __ballot(base + run > target), any = __ballot(m > 0.0);
        if (any != 0) full = k0 + 63 - __builtin_clzll(any);
        if (passed != 0) {
          const int f = __builtin_ctzll(passed);
          at = k0 + f;
          if (f > 0) base += lane_f64(run, f - 1);  // not run - m: rounded, that may pass the target
        } else {
          base += lane_f64(run, 63);
        }
      }
      const bool sought = at >= 0;  // else: a coin that no running sum passes; the last token that has mass
      if (!sought) at = full;
      if (tid == 0) {
        s_token = INT32_MAX;
        s_last = -1;
      }
      double r[NV][VEC];
      double mine = 0.0;
      int end = -1;  // the thread's last element that has mass
      const int v0 = at * unit + tid * NV;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float x[VEC];
        if (tid * NV + i < unit) {
          Row<T>::widen(row.load(v0 + i), x);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) x[k] = -INFINITY;
        }
        if constexpr (!kProbs) take_out<VEC>(x, row.first(v0 + i), rejected, static_cast<int>(token));
        residual<Q, VEC>(x, qrow, row.first(v0 + i), row.vocab, c, top, spent, r[i]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          mine += r[i][k];
          if (r[i][k] > 0.0) end = row.first(v0 + i) + k;
        }
      }
      double run = mine;
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) {
        const double o = __shfl_up(run, k, 64);
        if (lane >= k) run += o;
      }
      if (lane == 63) s_scan[wave] = run;
      __syncthreads();
      double from = base;
      for (int k = 0; k < wave; ++k) from += s_scan[k];
      const double left = __shfl_up(run, 1, 64);
      const double begin = lane == 0 ? from : from + left, stop = from + run;
      // A wave's first lane past the target: not only the one that the target lies in, as the scan's sums are rounded each in its
      // own order, and a lane without mass may seem to take the sum across it.
      const uint64_t past = __ballot(sought && stop > target && end >= 0);
      if (past != 0 && lane == __builtin_ctzll(past)) {
        double acc = begin;
        int hit = end;
        bool open = true;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            acc += r[i][k];
            if (open && acc > target && r[i][k] > 0.0) {
              hit = row.first(v0 + i) + k;
              open = false;
            }
          }
        atomicMin(&s_token, hit);
      }
      if (end >= 0) atomicMax(&s_last, end);
      __syncthreads();
      found = s_token != INT32_MAX ? s_token : (s_last >= 0 ? s_last : 0);
    }
    out_token(found);
    break;
  }
  for (int i = count + tid; i < a.width; i += kWalkThreads) a.sampled[b * a.stride_sampled + i] = -1;
  if (tid == 0) {
    state->stopped = 0;
    a.num_sampled[b] = count;
    if (slot >= 0 && slot < a.slots) a.path_len[slot] = count;
  }
}

Split split_of(const eagle4_sample_tree_args& a) {
  const int vec = a.dtype == EAGLE4_F32 ? 4 : 8;
  Split s;
  // a row may start up to vec - 1 elements behind a 16-byte boundary
  s.chunks = static_cast<int>(e4::ceil_div(e4::ceil_div(static_cast<int64_t>(a.vocab) + vec - 1, vec), kChunk / vec));
  const int64_t stats = a.rows * s.chunks;
  s.masses_off = stats * 8;
  s.state_off = s.masses_off + (a.probs != nullptr ? static_cast<int64_t>(a.num_reqs) * s.chunks * kParts * 8 : 0);
  s.maxes_off = s.state_off + static_cast<int64_t>(a.num_reqs) * static_cast<int64_t>(sizeof(State));
  return s;
}

int64_t workspace_of(const eagle4_sample_tree_args& a) {
  const Split s = split_of(a);
  return s.maxes_off + a.rows * s.chunks * 4;
}

bool tab_ok(const eagle4_itab& t) { return t.ptr != nullptr && e4::is_index_dtype(t.dtype); }

template <typename T, typename Q>
int launch(const eagle4_sample_tree_args& a, hipStream_t s) {
  const Split split = split_of(a);
  const int64_t stats = a.rows * split.chunks;
  if (stats >= 1 << 25) return EAGLE4_NOT_COVERED;  // 64 threads each: under 2^32
  const int pairs = a.probs == nullptr ? 0 : (a.width - 1 < kPairs ? a.width - 1 : kPairs);
  // Without draft probabilities a walk of many rows goes in two: the trees' first rows, then what is left of each tree under
  // the child that was accepted. Two launches more, but a fraction of the rows (64 requests, vocabulary 151936, trees of
  // 16 rows each, 39000 chunks: 95 instead of 135 us; trees of 8, 19000: 76 and 79; 16 requests, trees of 16, 9700: 58 and 51).
  const bool two = a.probs == nullptr && a.width > 1 && stats >= kTwoSteps;
  const auto chunks_of = [&](int rows, int first) {
    sample_chunks_of<T><<<dim3(e4::ceil_div(split.chunks, kWaves), rows, a.num_reqs), kThreads, 0, s>>>(a, split, first);
  };
  if (two)
    chunks_of(1, 1);
  else if (stats > 0)
    sample_chunks<T><<<e4::ceil_div(stats, kWaves), kThreads, 0, s>>>(a, split);
  sample_walk<T, Q><<<a.num_reqs, kWalkThreads, 0, s>>>(a, split, 1, pairs == 0, two);
  if (two) {
    chunks_of(a.width, 0);
    sample_walk<T, Q><<<a.num_reqs, kWalkThreads, 0, s>>>(a, split, 0, 1, 0);
  }
  if constexpr (Q::code >= 0) {
    for (int i = 1; i <= pairs; ++i) {
      sample_residual<T, Q><<<dim3(e4::ceil_div(split.chunks * kParts, kWaves), a.num_reqs), kThreads, 0, s>>>(a, split);
      sample_walk<T, Q><<<a.num_reqs, kWalkThreads, 0, s>>>(a, split, 0, i == pairs, 0);
    }
  }
  return E4_LAUNCH_STATUS();
}

template <typename T>
int launch_t(const eagle4_sample_tree_args& a, hipStream_t s) {
  if (a.probs == nullptr) return launch<T, NoQ>(a, s);
  switch (a.prob_dtype) {
    case EAGLE4_BF16: return launch<T, e4::Bf16>(a, s);
    case EAGLE4_F16: return launch<T, e4::F16>(a, s);
    case EAGLE4_F32: return launch<T, e4::F32>(a, s);
    default: return EAGLE4_NOT_COVERED;
  }
}

bool covered(const eagle4_sample_tree_args* a) {
  return a->num_reqs > 0 && a->num_reqs <= 65535 && a->rows >= 0 && a->vocab >= 1 && a->vocab <= (1 << 30) && a->width >= 1 &&
         a->width <= kMaxRows && a->slots >= 1;
}

}  // namespace

extern "C" int64_t eagle4_sample_tree_workspace(const eagle4_sample_tree_args* a) {
  return covered(a) ? workspace_of(*a) : -1;
}

extern "C" int eagle4_sample_tree(const eagle4_sample_tree_args* a, void* stream) {
  if (a->num_reqs == 0) return EAGLE4_OK;
  if (!covered(a) || a->workspace == nullptr || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0 ||
      a->workspace_bytes < workspace_of(*a) || !tab_ok(a->cu_num_logits) || !tab_ok(a->idx_mapping) || !tab_ok(a->parents) ||
      a->final_coins == nullptr || a->temperature == nullptr || a->sampled == nullptr || a->num_sampled == nullptr ||
      a->path == nullptr || a->path_len == nullptr)
    return EAGLE4_NOT_COVERED;
  // (of no rows nothing is read)
  if (a->rows > 0 && (a->logits == nullptr || a->coins == nullptr || !tab_ok(a->drafted))) return EAGLE4_NOT_COVERED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case EAGLE4_BF16: return launch_t<e4::Bf16>(*a, s);
    case EAGLE4_F16: return launch_t<e4::F16>(*a, s);
    case EAGLE4_F32: return launch_t<e4::F32>(*a, s);
    default: return EAGLE4_NOT_COVERED;
  }
}
