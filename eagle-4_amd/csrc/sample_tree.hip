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
// Decisions are comparisons, so everything that enters them is held in 64 bits: exp2 is a polynomial there (15 operations
// an element at the rate of 32-bit ones, against about 10 with the hardware's 32-bit exp2, whose error would flip one
// comparison in 10^7, and of a flat row's running sums far more).
//
// Only rows on the walk are read. One workgroup per request; a wave sums one contiguous region of the row, so that the
// regions' sums, which the walk needs for Z anyway, also lead the final token's search to one region.

#include "common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 2^x for x <= 0 in 64 bits: 2^f on [-1/2, 1/2] by its interpolant of degree 8 at the Chebyshev nodes (relative error
// 1.1e-12; 2^0 is 1 exactly), scaled by ldexp. Below -1100, and for the NaN of -inf * 0: 0.
E4_DEV double exp2_64(double x) {
  x = __builtin_fmax(x, -1100.0);
  const double n = __builtin_rint(x), f = x - n;
  double p = 0x1.63d12bb868a16p-20;
  p = __builtin_fma(p, f, 0x1.00dc4a539768ap-16);
  p = __builtin_fma(p, f, 0x1.4308ac8f571ecp-13);
  p = __builtin_fma(p, f, 0x1.5d8745a73511cp-10);
  p = __builtin_fma(p, f, 0x1.3b2ab718157d2p-7);
  p = __builtin_fma(p, f, 0x1.c6b08dd6fcf68p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff823d4dp-3);
  p = __builtin_fma(p, f, 0x1.62e42fef84cf5p-1);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, static_cast<int>(n));
}

struct NoQ {  // no draft probabilities
  using storage = uint16_t;
  static constexpr int code = -1;
  static E4_DEV float to_f32(storage) { return 0.f; }
};

// A row of the vocabulary as 16-byte vectors of the logits: vector v holds elements v * VEC - past .. + VEC - 1, `past` the
// elements by which the row starts behind a 16-byte boundary. A vector that is not wholly inside the row is read element by
// element, -inf outside.
template <typename T>
struct Row {
  using S = typename T::storage;
  static constexpr int VEC = 16 / static_cast<int>(sizeof(S));
  const S* p;
  int vocab, past, vectors;
  E4_DEV Row(const void* logits, int64_t row, int64_t stride, int vocab_) : vocab(vocab_) {
    p = static_cast<const S*>(logits) + row * stride;
    past = static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(S));
    vectors = (vocab + past + VEC - 1) / VEC;
  }
  E4_DEV int first(int v) const { return v * VEC - past; }
  E4_DEV bool inside(int v) const { return first(v) >= 0 && first(v) + VEC <= vocab; }
  E4_DEV u32x4 raw(int v) const {  // v wholly inside
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + first(v)));
  }
  E4_DEV static void widen(const u32x4& w, float (&x)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (sizeof(S) == 4)
        x[i] = __uint_as_float(w[i]);
      else
        x[i] = T::to_f32(static_cast<S>(w[i / 2] >> (16 * (i % 2))));
    }
  }
  E4_DEV void edge(int v, float (&x)[VEC]) const {
    const int e0 = first(v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = e0 + i >= 0 && e0 + i < vocab ? T::to_f32(p[e0 + i]) : -INFINITY;
  }
  E4_DEV void load(int v, float (&x)[VEC]) const {
    if (inside(v))
      widen(raw(v), x);
    else
      edge(v, x);
  }
};

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

E4_DEV double wave_sum(double x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m, 64);
  return x;
}

// (value, index) with the first index on ties; NaN is the largest value.
E4_DEV bool better(float v, int i, float bv, int bi) {
  const bool vn = v != v, bn = bv != bv;
  if (vn || bn) return vn && (!bn || i < bi);
  return v > bv || (v == bv && i < bi);
}

constexpr int kMaxRows = 64;

template <typename T, typename Q, int NT>
__global__ __launch_bounds__(NT) void sample_tree_kernel(const eagle4_sample_tree_args a) {
  constexpr int NW = NT / 64, VEC = Row<T>::VEC;
  constexpr bool kProbs = Q::code >= 0;
  __shared__ int s_parent[kMaxRows];
  __shared__ int64_t s_draft[kMaxRows];
  __shared__ float s_coin[kMaxRows];
  __shared__ int s_rejected[kMaxRows];  // tokens taken out of the residual (no draft probabilities)
  __shared__ float s_max[NW];
  __shared__ int s_arg[NW];
  __shared__ double s_p[NW], s_r[NW], s_scan[NW];  // a region's mass of p, of the residual; scan totals
  __shared__ int s_token, s_last;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

  const int64_t slot = e4::ld(a.idx_mapping, b);
  const int64_t start = e4::ld(a.cu_num_logits, b);
  const int64_t rows = e4::ld(a.cu_num_logits, b + 1) - start;
  const bool valid = slot >= 0 && slot < a.slots && start >= 0 && rows > 0 && start + rows <= a.rows;
  const int limit = !valid ? 0 : static_cast<int>(rows < a.width ? rows : a.width);
  const float temperature = a.temperature[b];
  const bool greedy = !(temperature > 0.f);
  const double c = 1.4426950408889634 / static_cast<double>(temperature);
  if (tid < limit) {
    s_parent[tid] = static_cast<int>(e4::ld(a.parents, slot, tid));
    s_draft[tid] = e4::ld(a.drafted, start + tid);
    s_coin[tid] = a.coins[start + tid];
  }
  __syncthreads();

  int node = 0, count = 0;
  for (int step = 0; step < limit; ++step) {
    const Row<T> row(a.logits, start + node, a.stride_row, a.vocab);
    const QRow<Q, VEC> qrow(a.probs, start + node, a.stride_prob, row.past);
    const int per = (row.vectors + NW - 1) / NW;
    const auto region = [&](int w, int& lo, int& hi) {
      lo = w * per < row.vectors ? w * per : row.vectors;
      hi = lo + per < row.vectors ? lo + per : row.vectors;
    };

    // the row's maximum and every region's mass, relative to it
    float top = -INFINITY;
    bool single = greedy;  // all mass on the argmax
    if (!greedy) {
      float m = -INFINITY;
      double sum = 0.0;
      const auto take = [&](const float (&x)[VEC]) {
        float vm = x[0];
#pragma unroll
        for (int i = 1; i < VEC; ++i) vm = __builtin_elementwise_maximum(vm, x[i]);
        if (!(vm <= m)) {
          sum *= exp2_64((static_cast<double>(m) - static_cast<double>(vm)) * c);
          m = vm;
        }
        const double off = -static_cast<double>(m) * c;
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum += exp2_64(__builtin_fma(static_cast<double>(x[i]), c, off));
      };
      int lo, hi;
      region(wave, lo, hi);
      for (int v = lo + lane; v < hi; v += 64) {
        float x[VEC];
        row.load(v, x);
        take(x);
      }
      float wm = m;
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) wm = __builtin_elementwise_maximum(wm, __shfl_xor(wm, k, 64));
      sum = wave_sum(sum * exp2_64((static_cast<double>(m) - static_cast<double>(wm)) * c));
      if (lane == 0) {
        s_max[wave] = wm;
        s_p[wave] = sum;
      }
      __syncthreads();
      top = s_max[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) top = __builtin_elementwise_maximum(top, s_max[w]);
      single = !(__builtin_fabsf(top) < INFINITY);
      if (!single && tid < NW)
        s_p[tid] *= exp2_64((static_cast<double>(s_max[tid]) - static_cast<double>(top)) * c);
      __syncthreads();
    }
    int arg = 0;
    if (single) {
      float bv = -INFINITY;
      int bi = INT32_MAX;
      for (int v = tid; v < row.vectors; v += NT) {
        float x[VEC];
        row.load(v, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int e = row.first(v) + i;
          if (e >= 0 && e < row.vocab && better(x[i], e, bv, bi)) {
            bv = x[i];
            bi = e;
          }
        }
      }
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) {
        const float ov = __shfl_xor(bv, k, 64);
        const int oi = __shfl_xor(bi, k, 64);
        if (better(ov, oi, bv, bi)) {
          bv = ov;
          bi = oi;
        }
      }
      if (lane == 0) {
        s_max[wave] = bv;
        s_arg[wave] = bi;
      }
      __syncthreads();
      bv = s_max[0];
      arg = s_arg[0];
      for (int w = 1; w < NW; ++w)
        if (better(s_max[w], s_arg[w], bv, arg)) {
          bv = s_max[w];
          arg = s_arg[w];
        }
      __syncthreads();
    }

    // exp2((l - top) c), the row's p times `total`
    const double off = -static_cast<double>(top) * c;
    const auto weight = [&](float l) { return exp2_64(__builtin_fma(static_cast<double>(l), c, off)); };
    double total = 0.0;
    if (!single) {
#pragma unroll
      for (int w = 0; w < NW; ++w) total += s_p[w];
    }
    double spent = 0.0, mass = total;  // s and Z, times `total`
    int rejected = 0;
    // the residual of a vector's elements, times `total`
    const auto residual = [&](int v, double (&r)[VEC]) {
      float x[VEC];
      row.load(v, x);
      if constexpr (kProbs) {
        float q[VEC];
        if (spent > 0.0) qrow.load(row.first(v), row.vocab, q);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          r[i] = weight(x[i]);
          if (spent > 0.0) r[i] = __builtin_fmax(r[i] - spent * static_cast<double>(q[i]), 0.0);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r[i] = weight(x[i]);
        for (int k = 0; k < rejected; ++k) {
          const int at = s_rejected[k] - row.first(v);
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (i == at) r[i] = 0.0;
        }
      }
    };
    const auto region_mass = [&](int w) {
      int lo, hi;
      region(w, lo, hi);
      double sum = 0.0;
      for (int v = lo + lane; v < hi; v += 64) {
        double r[VEC];
        residual(v, r);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum += r[i];
      }
      return wave_sum(sum);
    };

    // the children, in row order
    int next = -1;
    for (int child = 1; child < limit && next < 0; ++child) {
      if (s_parent[child] != node) continue;
      const int64_t token = s_draft[child];
      if (token < 0 || token >= row.vocab) continue;
      if (single) {
        if (token == arg) next = child;
        continue;
      }
      double r = weight(T::to_f32(row.p[token])), drawn = 1.0;
      if constexpr (kProbs) {
        drawn = static_cast<double>(Q::to_f32(qrow.p[token]));
        if (spent > 0.0) r = __builtin_fmax(r - spent * drawn, 0.0);
      } else {
        for (int k = 0; k < rejected; ++k)
          if (s_rejected[k] == token) r = 0.0;
      }
      if (static_cast<double>(s_coin[child]) * drawn * mass < r) {
        next = child;
      } else if constexpr (kProbs) {
        spent += mass;
        const double mine = region_mass(wave);
        __syncthreads();  // the last residual's masses have been read
        if (lane == 0) s_r[wave] = mine;
        __syncthreads();
        mass = 0.0;
#pragma unroll
        for (int w = 0; w < NW; ++w) mass += s_r[w];
      } else if (r > 0.0) {
        if (tid == 0) s_rejected[rejected] = static_cast<int>(token);
        ++rejected;
        mass = __builtin_fmax(mass - r, 0.0);
        __syncthreads();
      }
    }
    if (tid == 0) a.path[slot * a.stride_path + step] = node;
    ++count;
    if (next >= 0) {
      if (tid == 0) a.sampled[b * a.stride_sampled + step] = s_draft[next];
      node = next;
      __syncthreads();  // s_max, s_p, s_rejected have been read
      continue;
    }

    // no child accepted: the token of the final coin
    int64_t token = arg;
    if (!single) {
      if constexpr (!kProbs) {
        if (rejected > 0) {  // the regions that lost a token, summed again; the others' masses are p's
          int lo, hi;
          region(wave, lo, hi);
          bool lost = false;
          for (int k = 0; k < rejected; ++k) {
            const int v = (s_rejected[k] + row.past) / VEC;
            lost |= v >= lo && v < hi;
          }
          const double mine = lost ? region_mass(wave) : s_p[wave];
          if (lane == 0) s_r[wave] = mine;
          __syncthreads();
          mass = 0.0;
#pragma unroll
          for (int w = 0; w < NW; ++w) mass += s_r[w];
        }
      }
      bool whole = spent == 0.0 && rejected == 0;
      if (!whole && !(mass > 0.0)) {
        whole = true;
        spent = 0.0;
        rejected = 0;
        mass = total;
      }
      const double* const masses = whole ? s_p : s_r;
      const double target = static_cast<double>(a.final_coins[b]) * mass;
      double base = 0.0, before = 0.0;
      int at = -1, last = 0;
      bool sought = true;
      for (int w = 0; w < NW; ++w) {
        const double after = before + masses[w];
        if (masses[w] > 0.0) last = w;
        if (at < 0 && after > target) {
          at = w;
          base = before;
        }
        before = after;
      }
      if (at < 0) {  // a coin that no running sum passes: the last token that has mass
        at = last;
        sought = false;
      }
      if (tid == 0) {
        s_token = INT32_MAX;
        s_last = -1;
      }
      __syncthreads();
      int lo, hi;
      region(at, lo, hi);
      for (int v0 = lo; v0 < hi; v0 += NT) {
        const int v = v0 + tid;
        double r[VEC];
        double mine = 0.0;
        int end = -1;  // the last element that has mass
        if (v < hi) {
          residual(v, r);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            mine += r[i];
            if (r[i] > 0.0) end = row.first(v) + i;
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
        for (int w = 0; w < wave; ++w) from += s_scan[w];
        const double left = __shfl_up(run, 1, 64);
        const double begin = lane == 0 ? from : from + left, stop = from + run;
        if (sought && begin <= target && stop > target) {
          double acc = begin;
          int found = end;
          bool open = true;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            acc += r[i];
            if (open && acc > target && r[i] > 0.0) {
              found = row.first(v) + i;
              open = false;
            }
          }
          atomicMin(&s_token, found);
        }
        if (end >= 0) atomicMax(&s_last, end);
        for (int w = 0; w < NW; ++w) base += s_scan[w];
        __syncthreads();
        if (s_token != INT32_MAX) break;
      }
      token = s_token != INT32_MAX ? s_token : (s_last >= 0 ? s_last : 0);
    }
    if (tid == 0) a.sampled[b * a.stride_sampled + step] = token;
    break;
  }
  for (int i = count + tid; i < a.width; i += NT) a.sampled[b * a.stride_sampled + i] = -1;
  if (tid == 0) {
    a.num_sampled[b] = count;
    if (slot >= 0 && slot < a.slots) a.path_len[slot] = count;
  }
}

bool tab_ok(const eagle4_itab& t) { return t.ptr != nullptr && e4::is_index_dtype(t.dtype); }

template <typename T, typename Q>
int launch(const eagle4_sample_tree_args& a, hipStream_t s) {
  sample_tree_kernel<T, Q, 512><<<a.num_reqs, 512, 0, s>>>(a);
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

}  // namespace

extern "C" int eagle4_sample_tree(const eagle4_sample_tree_args* a, void* stream) {
  if (a->num_reqs == 0) return EAGLE4_OK;
  if (a->num_reqs < 0 || a->rows < 0 || a->vocab < 1 || a->vocab > (1 << 30) || a->width < 1 || a->width > kMaxRows ||
      a->slots < 1 || !tab_ok(a->drafted) || !tab_ok(a->cu_num_logits) || !tab_ok(a->idx_mapping) || !tab_ok(a->parents) ||
      a->coins == nullptr || a->final_coins == nullptr || a->temperature == nullptr || a->logits == nullptr)
    return EAGLE4_NOT_COVERED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case EAGLE4_BF16: return launch_t<e4::Bf16>(*a, s);
    case EAGLE4_F16: return launch_t<e4::F16>(*a, s);
    case EAGLE4_F32: return launch_t<e4::F32>(*a, s);
    default: return EAGLE4_NOT_COVERED;
  }
}
