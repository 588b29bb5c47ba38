// Rotary positions on gfx950: the first 2 `half` elements of every head of queries and keys, turned in pairs.
//
// Mathematics. The pair i of a head at position p, (x_i, x_{half + i}) or neighbours (x_{2i}, x_{2i + 1}), becomes
// (x c - y s, y c + x s), c and s the cosine and sine of p f_i times a factor. The angle is a product in 64 bits (in 32
// bits position 10^6 is off by 0.06 radians), taken to [-pi/4, pi/4] by two fused steps with pi/2 in two parts, and both
// series are summed there in 64 bits (Taylor's, to r^13 and r^14: the next terms are below 10^-13); c and s are rounded
// to 32 bits once. All heads of a token share them: a workgroup has them once in LDS, and
// nothing is read for them but f.
//
// A workgroup takes some tokens; a thread 16 bytes of a head, or the two 16-byte pieces whose elements are paired, several
// of them on their way together. What bounds it: HBM, one read and one write of each element: 8191 tokens of 32 and 8 heads of
// 128 (168 MB) take 34 us with their launch, 28 in a graph that finds part of them in the last cache; a copy's rate makes 33.
// 16 tokens take 4.8 us in a graph, a launch's latency and that of two loads after each other.

#include "common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int NT = 256;
constexpr int kAngles = 2048;  // of a workgroup, in LDS: 16 KB

E4_DEV void turn_of(double angle, double factor, float& c, float& s) {
  const double n = __builtin_rint(angle * 0.63661977236758134);  // 2 / pi
  double r = __builtin_fma(-n, 0x1.921fb54442d18p+0, angle);     // pi / 2, its first 53 bits
  r = __builtin_fma(-n, 0x1.1a62633145c07p-54, r);               // and the next
  const double z = r * r;
  double a = 1.0 / 6227020800.0;
  a = __builtin_fma(a, z, -1.0 / 39916800.0);
  a = __builtin_fma(a, z, 1.0 / 362880.0);
  a = __builtin_fma(a, z, -1.0 / 5040.0);
  a = __builtin_fma(a, z, 1.0 / 120.0);
  a = __builtin_fma(a, z, -1.0 / 6.0);
  a = __builtin_fma(a * z, r, r);
  double b = -1.0 / 87178291200.0;
  b = __builtin_fma(b, z, 1.0 / 479001600.0);
  b = __builtin_fma(b, z, -1.0 / 3628800.0);
  b = __builtin_fma(b, z, 1.0 / 40320.0);
  b = __builtin_fma(b, z, -1.0 / 720.0);
  b = __builtin_fma(b, z, 1.0 / 24.0);
  b = __builtin_fma(b, z, -0.5);
  b = __builtin_fma(b, z, 1.0);
  const int64_t quarter = static_cast<int64_t>(n);
  const double x = quarter & 1 ? -a : b, y = quarter & 1 ? b : a;  // a quarter turn on: (c, s) -> (-s, c)
  const double f = quarter & 2 ? -factor : factor;
  c = static_cast<float>(x * f);
  s = static_cast<float>(y * f);
}

template <typename T, int V>
struct Piece {  // V elements
  using S = typename T::storage;
  float x[V];
  E4_DEV void load(const S* p) {
    if constexpr (V == 1) {
      x[0] = T::to_f32(*p);
    } else {
      const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (sizeof(S) == 4)
          x[i] = __uint_as_float(w[i]);
        else
          x[i] = T::to_f32(static_cast<S>(w[i / 2] >> (16 * (i % 2))));
      }
    }
  }
  E4_DEV void store(S* p) const {
    if constexpr (V == 1) {
      *p = T::from_f32(x[0]);
    } else {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(S) == 4)
          w[i] = __float_as_uint(x[i]);
        else
          w[i] = T::pack(x[2 * i], x[2 * i + 1]);
      }
      *reinterpret_cast<u32x4*>(p) = w;
    }
  }
};

// The pieces of a head in the order of the threads: first the turned ones, then (not in place) the rest, copied as it is.
template <typename T, int V, bool kPaired>
__global__ __launch_bounds__(NT) void rotary_kernel(const eagle4_rotary_args a, int tokens_of, int pieces, int turned) {
  using S = typename T::storage;
  constexpr bool kTwo = !kPaired || V == 1;  // a turned unit is two pieces
  __shared__ float2 s_turn[kAngles];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens_of;
  const int tokens = static_cast<int>(a.tokens - first < tokens_of ? a.tokens - first : tokens_of);
  const int half = a.half;
  for (int i = threadIdx.x; i < tokens * half; i += NT) {
    const int t = i / half;
    float c, s;
    turn_of(static_cast<double>(e4::ld(a.positions, first + t)) * a.frequencies[i - t * half], a.factor, c, s);
    s_turn[i] = make_float2(c, s);
  }
  __syncthreads();
  const int heads = a.q_heads + a.k_heads;
  const uint32_t per_token = static_cast<uint32_t>(heads) * pieces, all = per_token * tokens;
  constexpr int U = 4;
  for (uint32_t u0 = threadIdx.x; u0 < all; u0 += U * NT) {
    Piece<T, V> x[U], y[U];
    S *to_x[U], *to_y[U];
    const float2* turn[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t unit = u0 + u * NT < all ? u0 + u * NT : u0;  // (past the last: the first again, not stored)
      const uint32_t t = unit / per_token, in = unit - t * per_token, h = in / pieces, piece = in - h * pieces;
      const bool key = h >= static_cast<uint32_t>(a.q_heads);
      const int64_t token = first + t, head = key ? h - a.q_heads : h;
      const S* from = static_cast<const S*>(key ? a.k : a.q) + token * (key ? a.stride_kt : a.stride_qt) +
                      head * (key ? a.stride_kh : a.stride_qh);
      S* to = static_cast<S*>(key ? a.k_out : a.q_out) + token * (key ? a.stride_kot : a.stride_qot) +
              head * (key ? a.stride_koh : a.stride_qoh);
      const bool turns = piece < static_cast<uint32_t>(turned);
      // a turned piece of neighbours is V / 2 pairs; else it has its pair's other piece beside it
      const int at = !turns ? 2 * half + (piece - turned) * V : kTwo && kPaired ? 2 * piece : piece * V;
      turn[u] = turns ? s_turn + t * half + (kPaired ? at / 2 : at) : nullptr;
      x[u].load(from + at);
      to_x[u] = to + at;
      to_y[u] = nullptr;
      if (kTwo && turns) {
        const int pair = kPaired ? at + 1 : half + at;
        y[u].load(from + pair);
        to_y[u] = to + pair;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u0 + u * NT >= all) continue;
      if (turn[u] != nullptr) {
        if constexpr (!kTwo) {
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            const float2 w = turn[u][i / 2];
            const float p = x[u].x[i], q = x[u].x[i + 1];
            x[u].x[i] = p * w.x - q * w.y;
            x[u].x[i + 1] = q * w.x + p * w.y;
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 w = turn[u][i];
            const float p = x[u].x[i], q = y[u].x[i];
            x[u].x[i] = p * w.x - q * w.y;
            y[u].x[i] = q * w.x + p * w.y;
          }
          y[u].store(to_y[u]);
        }
      }
      x[u].store(to_x[u]);
    }
  }
}

template <typename T, int V, bool kPaired>
int launch(const eagle4_rotary_args& a, hipStream_t s) {
  const bool in_place = (a.q_heads == 0 || a.q == a.q_out) && (a.k_heads == 0 || a.k == a.k_out);
  // neighbours one by one: a unit is a pair
  const int turned = kPaired && V > 1 ? 2 * a.half / V : a.half / V;
  const int pieces = turned + (in_place ? 0 : (a.dim - 2 * a.half) / V);
  // enough tokens for an angle a thread, and for four pieces a thread
  const int heads = a.q_heads + a.k_heads;
  int tokens_of = 1;
  while (2 * tokens_of * a.half <= kAngles && (tokens_of * a.half < NT || static_cast<int64_t>(heads) * pieces * tokens_of < 4 * NT) &&
         a.tokens > static_cast<int64_t>(512) * tokens_of)
    tokens_of *= 2;
  if (static_cast<int64_t>(heads) * pieces * tokens_of > (1 << 28)) return EAGLE4_NOT_COVERED;
  const int64_t grid = (a.tokens + tokens_of - 1) / tokens_of;
  if (grid >= (1 << 24)) return EAGLE4_NOT_COVERED;  // (256 threads each: under 2^32)
  rotary_kernel<T, V, kPaired><<<static_cast<unsigned>(grid), NT, 0, s>>>(a, tokens_of, pieces, turned);
  return E4_LAUNCH_STATUS();
}

template <typename T>
int launch_t(const eagle4_rotary_args& a, hipStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(typename T::storage));
  // 16-byte pieces where every head starts on 16 bytes and a piece is wholly turned or wholly not
  const auto on16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const auto whole = [](int64_t n) { return n % V == 0; };
  const bool q = a.q_heads == 0 || (on16(a.q) && on16(a.q_out) && whole(a.stride_qt) && whole(a.stride_qh) &&
                                    whole(a.stride_qot) && whole(a.stride_qoh));
  const bool k = a.k_heads == 0 || (on16(a.k) && on16(a.k_out) && whole(a.stride_kt) && whole(a.stride_kh) &&
                                    whole(a.stride_kot) && whole(a.stride_koh));
  const bool wide = q && k && whole(a.paired ? 2 * a.half : a.half) && whole(a.dim - 2 * a.half);
  if (a.paired) return wide ? launch<T, V, true>(a, s) : launch<T, 1, true>(a, s);
  return wide ? launch<T, V, false>(a, s) : launch<T, 1, false>(a, s);
}

}  // namespace

extern "C" int eagle4_rotary(const eagle4_rotary_args* a, void* stream) {
  if (a->tokens == 0 || (a->q_heads == 0 && a->k_heads == 0)) return EAGLE4_OK;
  if (a->tokens < 0 || a->tokens > (1 << 30) || a->q_heads < 0 || a->k_heads < 0 || a->half < 1 || a->half > 512 ||
      a->dim < 2 * a->half || a->dim > 1 << 16 || a->q_heads + static_cast<int64_t>(a->k_heads) > 4096 ||
      a->positions.ptr == nullptr || !e4::is_index_dtype(a->positions.dtype) || a->frequencies == nullptr ||
      (a->q_heads > 0 && (a->q == nullptr || a->q_out == nullptr)) || (a->k_heads > 0 && (a->k == nullptr || a->k_out == nullptr)))
    return EAGLE4_NOT_COVERED;
  // in place together, or not: the rest of a head is copied for both or for neither
  if (a->q_heads > 0 && a->k_heads > 0 && (a->q == a->q_out) != (a->k == a->k_out)) return EAGLE4_NOT_COVERED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case EAGLE4_BF16: return launch_t<e4::Bf16>(*a, s);
    case EAGLE4_F16: return launch_t<e4::F16>(*a, s);
    case EAGLE4_F32: return launch_t<e4::F32>(*a, s);
    default: return EAGLE4_NOT_COVERED;
  }
}
