// Rows quantised into fp8-e4m3 pages with one scale per (page, head), and gathered back, on gfx950.
//
// Mathematics. A page's scale s is a power of two, the least with amax <= 448 s over the page's rows: value x is held as
// e4m3(x / s). e4m3 is a floating format, so its relative error (2^-4) is the same at any scale and a power of two costs
// no precision against amax / 448; x / s is exact, so each value is rounded once, and when later rows make a page's scale
// grow by 2^k its earlier rows move by k binades: exact but where they leave e4m3's normal range (below 2^-6 of the new
// scale), as those values lie there in any case. The earlier rows of a page (positions below the context) are re-encoded
// only when the scale grows; a page that starts at or after the context starts afresh, whatever it held.
//
// Both directions are bound by HBM where there is much to move, and by one chain of dependent loads (lengths, page
// table, rows, scale) where there is little. Measured (bf16 rows): 4 prompts of 8 heads x 128, K and V, written in 22 us (3.3
// TB/s read and written, latency's more than HBM's: each wave's chain is five loads long, and 28 waves a CU hide most of
// it); 64 rounds' accepted rows in 6.3 us, nearly all of it that chain and the launch; 8 long requests read in 35 us where
// half of the pages lie in the last-level cache, as in a replay (5.7 TB/s read and written, 32 of 66 MB from HBM; with one
// chunk a lane in flight 56 us), and in 45 us from cold caches (4.4 TB/s; a copy of 1 GiB reaches 5.15); one latent request in
// 5.2 us.

#include "common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kMaxE4m3 = 448.f;

// The least power of two s with amax <= 448 s (448 = 1.75 * 2^8), by its bits; at least 2^-126, 0 for 0.
E4_DEV float page_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  if (bits == 0) return 0.f;
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(e < 1 ? 1 : e) << 23);
}

// Two values of magnitude at most 448 (or NaN) rounded to e4m3, nearest even.
E4_DEV uint32_t encode2(float x, float y) {
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false)) & 0xffffu;
}
// x / s as e4m3 takes it: an infinity saturates, NaN stays.
E4_DEV float scaled(float x, float inv) {
  const float y = x * inv;
  return __builtin_fabsf(x) == INFINITY ? __builtin_copysignf(kMaxE4m3, x) : y;
}
E4_DEV float finite_abs(float x) {
  const float a = __builtin_fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// N values in fp8 (N 8: one 8-byte load), widened, and back.
template <int N>
struct Codes {
  u32x2 w;
  E4_DEV void load(const uint8_t* p) {
    if constexpr (N == 8)
      w = *reinterpret_cast<const u32x2*>(p);
    else
      w[0] = *p;
  }
  E4_DEV void widen(float (&x)[N]) const {
    if constexpr (N == 8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
        x[4 * i] = lo[0];
        x[4 * i + 1] = lo[1];
        x[4 * i + 2] = hi[0];
        x[4 * i + 3] = hi[1];
      }
    } else {
      x[0] = __builtin_amdgcn_cvt_pk_f32_fp8(w[0], false)[0];
    }
  }
};
template <int N>
E4_DEV void store_codes(uint8_t* p, const float (&x)[N]) {
  if constexpr (N == 8) {
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = encode2(x[4 * i], x[4 * i + 1]) | encode2(x[4 * i + 2], x[4 * i + 3]) << 16;
    *reinterpret_cast<u32x2*>(p) = w;
  } else {
    *p = static_cast<uint8_t>(encode2(x[0], 0.f));
  }
}

// A chunk of N elements (8: 16-byte loads) of dtype T as loaded, and widened.
template <typename T, int N>
struct Chunk {
  static constexpr int kWords = N * static_cast<int>(sizeof(typename T::storage)) / 4;
  u32x4 w[N == 8 ? kWords / 4 : 1];
  E4_DEV void load(const typename T::storage* p) {
    if constexpr (N == 8) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) w[i] = reinterpret_cast<const u32x4*>(p)[i];
    } else if constexpr (sizeof(typename T::storage) == 4) {
      w[0][0] = __float_as_uint(*p);
    } else {
      w[0][0] = *p;
    }
  }
  E4_DEV void widen(float (&x)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (sizeof(typename T::storage) == 4)
        x[i] = __uint_as_float(w[i / 4][i % 4]);
      else
        x[i] = T::to_f32(static_cast<uint16_t>(w[0][i / 2] >> (16 * (i % 2))));
    }
  }
};

// A position's page; the division is a 32-bit one for all but the longest.
E4_DEV int64_t page_of(int64_t position, int page) {
  if (position >> 32 == 0) return static_cast<uint32_t>(position) / static_cast<uint32_t>(page);
  return position / page;
}

// One wave per (matrix, head, page, request); waves of a workgroup take adjacent heads. `pages`: pages a request's rows can
// reach at most. The page's rows stay in registers between the maximum and the rounding where they fit in kHeld chunks a
// lane (16 rows of 256 elements), else they are read twice.
template <typename T, int N, int kHeld>
__global__ __launch_bounds__(256) void write_kernel(const eagle4_write_kv_args a, int pages) {
  using S = typename T::storage;
  const int lane = threadIdx.x & 63;
  const int item = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int matrices = a.value != nullptr ? 2 : 1;
  const int p = item / (a.heads * matrices), hm = item % (a.heads * matrices);
  const int head = hm % a.heads, b = blockIdx.y;
  const bool second = hm >= a.heads;
  if (p >= pages) return;

  const int64_t context = e4::ld(a.context_lens, b);
  const int64_t start = e4::ld(a.query_start_loc, b);
  const int64_t end = e4::ld(a.query_start_loc, b + 1);
  int64_t slot = 0, count = end - start;
  if (a.path.ptr != nullptr) {
    slot = e4::ld(a.idx_mapping, b);
    if (slot < 0 || slot >= a.path_slots) return;
    count = e4::ld(a.path_len, slot);
    count = count < a.path_width ? count : a.path_width;
  }
  count = count < a.max_rows ? count : a.max_rows;
  if (context < 0 || count <= 0 || start < 0 || end > a.tokens) return;
  const int64_t index = page_of(context, a.page) + p, first = index * a.page;
  const int64_t lo = first > context ? first : context;
  const int64_t hi = first + a.page < context + count ? first + a.page : context + count;
  if (lo >= hi || index >= a.max_blocks) return;
  const int64_t block = e4::ld(a.block_table, b, index);
  if (block < 0 || block >= a.num_blocks) return;

  const S* const src = static_cast<const S*>(second ? a.value : a.key) + head * (second ? a.stride_vh : a.stride_kh);
  const int64_t stride_row = second ? a.stride_vt : a.stride_kt;
  uint8_t* const dst = static_cast<uint8_t*>(second ? a.value_cache : a.key_cache) +
                       block * (second ? a.stride_vcb : a.stride_kcb) + head * (second ? a.stride_vch : a.stride_kch);
  const int64_t stride_slot = second ? a.stride_vcs : a.stride_kcs;
  float* const scale = (second ? a.v_scale : a.k_scale) + block * (second ? a.stride_vsb : a.stride_ksb) +
                       head * (second ? a.stride_vsh : a.stride_ksh);
  const float held_scale = *scale;

  const int per_row = a.dim / N, rows = static_cast<int>(hi - lo), chunks = rows * per_row;
  // the source of chunk c; null where the path names no row of the request
  auto source = [&](int c) -> const S* {
    const int r = c / per_row, col = (c - r * per_row) * N;
    const int64_t j = lo - context + r;
    const int64_t row = a.path.ptr != nullptr ? e4::ld(a.path, slot, j) : j;
    if (row < 0 || row >= end - start) return nullptr;
    return src + (start + row) * stride_row + col;
  };
  Chunk<T, N> held[kHeld];
  const S* from[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int c = lane + 64 * i;
    from[i] = c < chunks ? source(c) : nullptr;
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (from[i] != nullptr) held[i].load(from[i]);
  float amax = 0.f;
  bool any = false;  // a row goes to the page
  auto most = [&](const Chunk<T, N>& ch) {
    any = true;
    float x[N];
    ch.widen(x);
#pragma unroll
    for (int i = 0; i < N; ++i) amax = fmaxf(amax, finite_abs(x[i]));
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (from[i] != nullptr) most(held[i]);
  for (int c = lane + 64 * kHeld; c < chunks; c += 64) {
    const S* const s = source(c);
    if (s == nullptr) continue;
    Chunk<T, N> ch;
    ch.load(s);
    most(ch);
  }
  if (!__any(any)) return;  // (a request padded into the batch has another's path and no rows: the page is not its own)
  amax = e4::group_max<64>(amax);
  // Whether the rows hold an infinity: looked for only where no other value gives the page a scale.
  auto infinite = [&] {
    bool inf = false;
    auto look = [&](const Chunk<T, N>& ch) {
      float x[N];
      ch.widen(x);
#pragma unroll
      for (int i = 0; i < N; ++i) inf = inf || __builtin_fabsf(x[i]) == INFINITY;
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (from[i] != nullptr) look(held[i]);
    for (int c = lane + 64 * kHeld; c < chunks; c += 64) {
      const S* const s = source(c);
      if (s == nullptr) continue;
      Chunk<T, N> ch;
      ch.load(s);
      look(ch);
    }
    return __any(inf) != 0;
  };

  const int kept = static_cast<int>(lo - first);  // earlier rows of the page
  const float old = kept > 0 ? held_scale : 0.f;
  float now = fmaxf(old, page_scale(amax));
  if (now == 0.f && infinite()) now = 1.f;  // else they would read back as zeros
  const float inv = now > 0.f ? 1.0f / now : 0.f;
  if (kept > 0 && now > old) {
    const float ratio = old * inv;
    for (int c = lane; c < kept * per_row; c += 64) {
      const int r = c / per_row, col = (c - r * per_row) * N;
      float x[N];
      Codes<N> codes;
      codes.load(dst + r * stride_slot + col);
      codes.widen(x);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] *= ratio;
      store_codes<N>(dst + r * stride_slot + col, x);
    }
  }
  auto put = [&](const Chunk<T, N>& ch, int c) {
    const int r = c / per_row, col = (c - r * per_row) * N;
    float x[N];
    ch.widen(x);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = scaled(x[i], inv);
    store_codes<N>(dst + (kept + r) * stride_slot + col, x);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (from[i] != nullptr) put(held[i], lane + 64 * i);
  for (int c = lane + 64 * kHeld; c < chunks; c += 64) {
    const S* const s = source(c);
    if (s == nullptr) continue;
    Chunk<T, N> ch;
    ch.load(s);
    put(ch, c);
  }
  if (lane == 0) *scale = now;
}

// One workgroup per (run of `rows` positions, request, matrix), all heads. kAhead chunks of N elements a lane are on their way
// together: table entries, then codes and scales, then the stores. A page that the table does not have (or names out of
// range) reads as zeros.
template <typename T, int N>
__global__ __launch_bounds__(256) void read_kernel(const eagle4_read_kv_args a, int rows) {
  using S = typename T::storage;
  constexpr int kAhead = 4;
  const int b = blockIdx.y;
  const bool second = blockIdx.z != 0;
  const int64_t start = e4::ld(a.start_loc, b), end = e4::ld(a.start_loc, b + 1);
  const int lo = static_cast<int>(blockIdx.x) * rows;
  if (start < 0 || end > a.tokens || lo >= end - start || lo >= a.max_len) return;
  const int64_t most = end - start < a.max_len ? end - start : a.max_len;
  const int n = static_cast<int>(most - lo < rows ? most - lo : rows);
  const int per_head = a.dim / N, per_row = per_head * a.heads, total = n * per_row;
  const uint8_t* const cache = static_cast<const uint8_t*>(second ? a.value_cache : a.key_cache);
  const int64_t stride_block = second ? a.stride_vcb : a.stride_kcb, stride_slot = second ? a.stride_vcs : a.stride_kcs,
                stride_head = second ? a.stride_vch : a.stride_kch;
  const float* const scales = second ? a.v_scale : a.k_scale;
  const int64_t stride_sb = second ? a.stride_vsb : a.stride_ksb, stride_sh = second ? a.stride_vsh : a.stride_ksh;
  S* const rows_out = static_cast<S*>(second ? a.value : a.key) + (start + lo) * (second ? a.stride_vt : a.stride_kt);
  const int64_t stride_t = second ? a.stride_vt : a.stride_kt, stride_h = second ? a.stride_vh : a.stride_kh;
  // chunk c is row c / per_row; the lane's next one is 256 on
  const int step_row = 256 / per_row, step_col = 256 % per_row;
  int r = static_cast<int>(threadIdx.x) / per_row, hc = static_cast<int>(threadIdx.x) % per_row;
  for (int c0 = threadIdx.x; c0 < total; c0 += 256 * kAhead) {
    int64_t block[kAhead];
    int row[kAhead], head[kAhead], col[kAhead], slot[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      row[i] = r;
      head[i] = static_cast<int>(static_cast<uint32_t>(hc) / static_cast<uint32_t>(per_head));
      col[i] = (hc - head[i] * per_head) * N;
      const int index = static_cast<int>(static_cast<uint32_t>(lo + r) / static_cast<uint32_t>(a.page));
      slot[i] = lo + r - index * a.page;
      block[i] = c0 + 256 * i < total && index < a.max_blocks ? e4::ld(a.block_table, b, index) : -1;
      r += step_row;
      hc += step_col;
      if (hc >= per_row) {
        hc -= per_row;
        ++r;
      }
    }
    Codes<N> codes[kAhead];
    float s[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      s[i] = 0.f;
      codes[i] = Codes<N>{};
      if (block[i] >= 0 && block[i] < a.num_blocks) {
        codes[i].load(cache + block[i] * stride_block + slot[i] * stride_slot + head[i] * stride_head + col[i]);
        s[i] = scales[block[i] * stride_sb + head[i] * stride_sh];
      } else {
        block[i] = -1;
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (c0 + 256 * i >= total) break;
      float x[N];
      codes[i].widen(x);
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = block[i] < 0 ? 0.f : x[k] * s[i];
      S* const out = rows_out + row[i] * stride_t + head[i] * stride_h + col[i];
      if constexpr (N == 8) {
        constexpr int kVecs = static_cast<int>(sizeof(S)) / 2;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          u32x4 w;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (sizeof(S) == 4)
              w[k] = __float_as_uint(x[4 * v + k]);
            else
              w[k] = T::pack(x[2 * k], x[2 * k + 1]);
          }
          reinterpret_cast<u32x4*>(out)[v] = w;
        }
      } else {
        *out = T::from_f32(x[0]);
      }
    }
  }
}

bool tab_ok(const eagle4_itab& t) { return t.ptr != nullptr && e4::is_index_dtype(t.dtype); }
bool multiple(int64_t v, int64_t of) { return v % of == 0; }
bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Whether rows and pages can be moved eight elements at a time.
template <typename A>
bool vectors(const A& a) {
  const bool v = a.value != nullptr;
  for (const int64_t s : {int64_t(a.dim), a.stride_kt, a.stride_kh, a.stride_kcb, a.stride_kcs, a.stride_kch,
                          v ? a.stride_vt : 0, v ? a.stride_vh : 0, v ? a.stride_vcb : 0, v ? a.stride_vcs : 0,
                          v ? a.stride_vch : 0})
    if (!multiple(s, 8)) return false;
  return aligned(a.key, 16) && aligned(a.key_cache, 8) && (!v || (aligned(a.value, 16) && aligned(a.value_cache, 8)));
}

template <typename A>
bool pages_ok(const A& a) {
  return (a.key != nullptr || a.tokens == 0) && a.key_cache != nullptr && a.k_scale != nullptr &&
         (a.value == nullptr || (a.value_cache != nullptr && a.v_scale != nullptr)) && tab_ok(a.block_table) &&
         a.heads > 0 && a.dim > 0 && a.page > 0 && a.max_blocks >= 0 && a.num_blocks >= 0 && a.num_reqs <= 65535 &&
         int64_t(a.heads) * a.dim <= (1 << 20) && int64_t(a.dim) * a.page <= (1 << 24);
}

template <typename T>
int launch_write(const eagle4_write_kv_args& a, hipStream_t s) {
  // rows from any slot of a first page on reach at most this many pages
  const int pages = e4::ceil_div(int64_t(a.max_rows) - 1, a.page) + 1;
  const int64_t items = int64_t(pages) * a.heads * (a.value != nullptr ? 2 : 1);
  if (items > (int64_t(1) << 30)) return EAGLE4_NOT_COVERED;
  const dim3 grid(e4::ceil_div(items, 4), a.num_reqs);
  // where a page's rows fit four chunks a lane, twice the waves fit a CU (72 registers instead of 108): 22.0 instead of
  // 24.7 us for 4 prompts of 16 x 128 pages
  if (!vectors(a))
    write_kernel<T, 1, 4><<<grid, 256, 0, s>>>(a, pages);
  else if (int64_t(a.page) * a.dim <= 4 * 64 * 8)
    write_kernel<T, 8, 4><<<grid, 256, 0, s>>>(a, pages);
  else
    write_kernel<T, 8, 8><<<grid, 256, 0, s>>>(a, pages);
  return E4_LAUNCH_STATUS();
}

template <typename T>
int launch_read(const eagle4_read_kv_args& a, hipStream_t s) {
  const int rows = 16;
  const dim3 grid(e4::ceil_div(a.max_len, rows), a.num_reqs, a.value != nullptr ? 2 : 1);
  if (vectors(a))
    read_kernel<T, 8><<<grid, 256, 0, s>>>(a, rows);
  else
    read_kernel<T, 1><<<grid, 256, 0, s>>>(a, rows);
  return E4_LAUNCH_STATUS();
}

}  // namespace

extern "C" int eagle4_write_kv_pages(const eagle4_write_kv_args* a, void* stream) {
  if (a->num_reqs == 0 || a->max_rows <= 0) return EAGLE4_OK;
  if (!pages_ok(*a) || a->num_reqs < 0 || !tab_ok(a->context_lens) || !tab_ok(a->query_start_loc)) return EAGLE4_NOT_COVERED;
  if (a->path.ptr != nullptr && (!tab_ok(a->path) || !tab_ok(a->path_len) || !tab_ok(a->idx_mapping)))
    return EAGLE4_NOT_COVERED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case EAGLE4_BF16: return launch_write<e4::Bf16>(*a, s);
    case EAGLE4_F16: return launch_write<e4::F16>(*a, s);
    case EAGLE4_F32: return launch_write<e4::F32>(*a, s);
    default: return EAGLE4_NOT_COVERED;
  }
}

extern "C" int eagle4_read_kv_pages(const eagle4_read_kv_args* a, void* stream) {
  if (a->num_reqs == 0 || a->max_len <= 0) return EAGLE4_OK;
  if (!pages_ok(*a) || a->num_reqs < 0 || !tab_ok(a->start_loc)) return EAGLE4_NOT_COVERED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case EAGLE4_BF16: return launch_read<e4::Bf16>(*a, s);
    case EAGLE4_F16: return launch_read<e4::F16>(*a, s);
    case EAGLE4_F32: return launch_read<e4::F32>(*a, s);
    default: return EAGLE4_NOT_COVERED;
  }
}
