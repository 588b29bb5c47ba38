// Rows of logits on gfx950: their 16-byte vectors, the weights of a softmax in 64 bits, reductions over a wave's lanes.
#pragma once

#include "common.h"

namespace e4vocab {

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
  E4_DEV u32x4 load(int v) const {
    if (inside(v)) return raw(v);
    const int e0 = first(v);
    u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const S x = e0 + i >= 0 && e0 + i < vocab ? p[e0 + i] : T::from_f32(-INFINITY);
      if constexpr (sizeof(S) == 4)
        w[i] = __float_as_uint(x);
      else
        w[i / 2] |= static_cast<uint32_t>(x) << (16 * (i % 2));
    }
    return w;
  }
};

// A value of another lane of the same 16, by a DPP pattern; of 64 bits in two halves.
template <int kCtrl>
E4_DEV double dpp64(double x) {
  const uint64_t w = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_mov_dpp(static_cast<int>(w), kCtrl, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_mov_dpp(static_cast<int>(w >> 32), kCtrl, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
// The sum with lane ^ 16 or lane ^ 32: swaps of rows of lanes.
template <int N>
E4_DEV double add_row(double x) {
  const uint64_t w = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = static_cast<uint32_t>(w), hi = static_cast<uint32_t>(w >> 32);
  const auto a = N == 16 ? __builtin_amdgcn_permlane16_swap(lo, lo, false, false) : __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
  const auto b = N == 16 ? __builtin_amdgcn_permlane16_swap(hi, hi, false, false) : __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(b[0]) << 32) | a[0]) +
         __builtin_bit_cast(double, (static_cast<uint64_t>(b[1]) << 32) | a[1]);
}
E4_DEV double sum16(double x) {  // over the 16 lanes of a row: lane ^ 1, ^ 2, the other quad, the other eight
  x += dpp64<0xB1>(x);
  x += dpp64<0x4E>(x);
  x += dpp64<0x141>(x);
  return x + dpp64<0x140>(x);
}
E4_DEV double wave_sum(double x) { return add_row<32>(add_row<16>(sum16(x))); }

E4_DEV float max16(float x) {  // NaN the largest
  x = __builtin_elementwise_maximum(x, e4::dpp<0xB1>(x));
  x = __builtin_elementwise_maximum(x, e4::dpp<0x4E>(x));
  x = __builtin_elementwise_maximum(x, e4::dpp<0x141>(x));
  return __builtin_elementwise_maximum(x, e4::dpp<0x140>(x));
}
E4_DEV float wave_max(float x) {
  const uint32_t w = __float_as_uint(max16(x));
  const auto a = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  const uint32_t v = __float_as_uint(__builtin_elementwise_maximum(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_elementwise_maximum(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

E4_DEV double scale_of(float temperature) { return 1.4426950408889634 / static_cast<double>(temperature); }
// exp2((x - top) c), exactly 1 at the maximum: the difference of two logits is taken before it is scaled. (One fma of x c and
// a rounded -top c would be an operation less, but its error is 2^-53 of |top| c: from 2^53 on, as with logits of a type's
// lowest value or temperatures below 1e-15, that is no error but the result.)
E4_DEV double weight_of(float x, float top, double c) {
  return exp2_64((static_cast<double>(x) - static_cast<double>(top)) * c);
}

}  // namespace e4vocab
