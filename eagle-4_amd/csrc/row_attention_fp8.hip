// Attention of decode-time draft rows (row_attention.hip) over fp8-e4m3 pages with a scale per (page, KV head), on gfx950.
//
// Mathematics. A row's key j, of its page's scales k_j and v_j, has the score s_j = scale k_j (q . K_j) and the value v_j V_j, K_j and
// V_j the codes, which the products take exactly (every e4m3 value is a bf16 and an fp16 value). With logarithms to base 2
// and t_j = s_j + log2 v_j, the weights are w_j = 2^(t_j - m), m a running maximum of t:
//     out = sum w_j V_j / sum w_j / v_j.
// So what is rounded for the second product is at most 2^kSlack and its largest terms are near 1; sums, maxima and the denominator
// are in 32 bits. Bf16 rows round a weight once to bf16 (2^-8 of it, as the output is rounded anyway). fp16 has not the range:
// a key without values (zeros under a large scale, or a page of scale 0, which counts as 1 here) may hold the maximum, and the weights
// that matter lie 2^-20 and more below it. So fp16 rows take each weight as two bf16 parts, 16 bits of it over the range of 32-bit floats;
// codes are bf16 values too. That costs 1 to 3% of a step, 2 to 15% of an extend (36 rows a head of D 128 over 2048 keys, 32 requests: 47
// -> 53 us; bf16 rows would pay as much, 47 -> 54). A page whose value scale is 0, or below 2^-100, counts in the denominator alone
// (its codes are taken as zeros). The keys that a row does not see weigh 0, and in tiles that hold such keys NaN codes are taken
// out of the values first (0 times NaN): they are added to the rows that see them.
//
// Split: a workgroup takes a key split (or the ancestors) of a request's KV head and up to 16 RT of its rows (request rows x
// query heads of the group); its four waves take every fourth tile of 32 keys on their own, each with its own softmax, and
// join at the end: no barrier is in the loop. K goes from memory into the registers that the matrix instructions read: a
// lane takes 16 bytes of its key, which are two steps of the product (the queries, in LDS, are read in that order of d). V has to be
// transposed and goes through the wave's own LDS. The next tile's loads start when this tile's K is used up and its V is in LDS, so
// one set of registers does; page entries are looked up a tile further ahead. Splits are joined by a second kernel.

#include "attention_tile.h"

namespace {

using namespace e4attn;

constexpr int NW = 4, NT = 64 * NW;
constexpr float kSlack = 8.f;

E4_DEV int64_t window_start(int64_t pos, int window) {
  if (window <= 0) return 0;
  const int64_t s = pos - window + 1;
  return s > 0 ? s : 0;
}

E4_DEV uint2 lds_tr8(const char* p) {
  typedef int v2i32 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i32*)p));
}

// The bytes of w that hold an e4m3 NaN (0x7f, 0xff), as 0x80 each.
E4_DEV uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// A value as one that the compiler knows nothing of: addresses made from it are made where they are used, and not kept in registers
// over the loop.
E4_DEV int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

struct WaveMeta {
  int64_t koff[32], voff[32];  // byte offsets of the tile's key and value rows
  float ks[32], lv[32], iv[32];  // scale log2(e) k_j, log2 v_j, 1 / v_j
};

template <int D, int RT>
struct Smem {
  static constexpr int kHalves = D >= 128 ? 2 : 1;  // the join takes the columns in so many parts
  union {
    struct {
      char q[RT * 16 * 2 * D];  // the rows, 16-byte chunks swizzled as Tile's keys
      char v[NW][32 * D];       // a wave's tile of values, rows of D codes in 16-byte chunks swizzled as Tile8's
      WaveMeta meta[NW];
      int2 seen[RT * 16];  // the first and the last key that a row sees
    } loop;
    struct {
      f32x4_t acc[NW][D / 16 / kHalves][64];
      float m[NW][RT * 16], l[NW][RT * 16];
    } join;
  };
};

// Waves a SIMD that the registers are kept for: the loads of one wave's tile do not cover its latency.
template <int D, int RT>
constexpr int kResident = D * RT <= 64 ? 5 : D * RT <= 128 ? 4 : D == 128 && RT == 2 ? 3 : 2;

template <int D, typename T, int RT>
__global__ __launch_bounds__(NT, (kResident<D, RT>)) void row_attention_fp8_kernel(const eagle4_row_attn_fp8_args x, int groups, int splits) {
  const eagle4_row_attn_args& a = x.rows;
  using T8 = Tile8<D>;
  constexpr int kParts = T::code == EAGLE4_F16 ? 2 : 1;  // of a weight, in bf16
  constexpr bool kEarly = D * RT <= 256;  // the next loads before the softmax; else behind it, for the registers
  constexpr int CH = D / 16, KJ = D / 64, NI = D / 32, RPI = 1024 / D;
  __shared__ __attribute__((aligned(1024))) Smem<D, RT> sm;
  // The row groups of a unit (a split of a request's KV head) run on one XCD (workgroup i on XCD i % 8) one after another, so that
  // its second one finds the keys in that XCD's cache; rows of units over the XCDs are skewed, so that no XCD has the same head
  // every time (its rows lie in a part of the cache's channels).
  const uint32_t at_xcd = blockIdx.x / 8u, turn = at_xcd / groups;
  const uint32_t unit = turn * 8u + ((blockIdx.x + turn) & 7u);
  if (unit >= static_cast<uint32_t>(splits) * a.kv_heads * a.bs) return;
  const int grp = at_xcd % groups, split = unit % splits, kvh = unit / splits % a.kv_heads, b = unit / splits / a.kv_heads;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int G = a.heads / a.kv_heads, R = a.rows_per_request * G;
  const bool extend = a.step == 0;
  const int NS = extend ? splits : splits - 1;  // of the shared range; a draft step's ancestors are one more
  int64_t seq_len = e4::ld(a.seq_lens, b);
  // Keys end with the page table: a row past it sees those before. (A padded request's length may be anything; far out it makes no
  // difference which.)
  const int64_t room = static_cast<int64_t>(x.table_width) * a.table_page, out = int64_t{1} << 32;
  seq_len = seq_len < -out ? -out : seq_len < room + out ? seq_len : room + out;
  int64_t trow = a.table_rows.ptr != nullptr ? e4::ld(a.table_rows, b) : b;
  trow = trow < 0 ? 0 : trow < x.table_height ? trow : x.table_height - 1;
  const int32_t* const table = a.table + trow * a.stride_table;

  // the queries of all rows go to LDS
  {
    constexpr int QC = D / 8, ALL = RT * 16 * QC;
#pragma unroll
    for (int i = 0; i < (ALL + NT - 1) / NT; ++i) {
      const int at = tid + i * NT, row = at / QC, chunk = at % QC, rho = grp * RT * 16 + row;
      if (ALL % NT != 0 && at >= ALL) break;
      const uint16_t* const p = static_cast<const uint16_t*>(a.q) +
                                (static_cast<int64_t>(b) * a.rows_per_request + rho / G) * a.stride_q_row +
                                static_cast<int64_t>(kvh * G + rho % G) * a.stride_q_head + 8 * chunk;
      u32x4_t w = {0u, 0u, 0u, 0u};
      if (rho < R) w = *reinterpret_cast<const u32x4_t*>(p);
      *reinterpret_cast<u32x4_t*>(sm.loop.q + row * 2 * D + 16 * (chunk ^ Tile<D>::kswz(row))) = w;
    }
  }

  // The split's keys: `count` positions from `start` on, or the rows' ancestor columns; row r sees keys lo[r] .. hi[r] of
  // them, and every row sees all_lo .. all_hi.
  const bool anc = !extend && split == NS;
  int64_t start = 0;
  int count = 0, all_lo = 0, all_hi = -1;
  int64_t end = 0;
  const auto within = [&](int64_t p) { return static_cast<int>(p < start - 1 ? -1 : p < end ? p - start : end - start); };
  if (!anc) {
    const int64_t first = window_start(extend ? seq_len : seq_len - 1, a.window);
    const int64_t newest = extend ? seq_len + a.rows_per_request - 1 : seq_len - 1, last = newest < room ? newest : room - 1;
    const int64_t span = last + 1 - first;
    const int64_t per = span > 0 ? ((span + NS - 1) / NS + 31) / 32 * 32 : 0;
    start = first + split * per;
    end = start + per < last + 1 ? start + per : last + 1;
    count = end > start ? static_cast<int>(end - start) : 0;
    all_lo = extend ? within(window_start(newest, a.window)) : 0;
    all_hi = extend ? within(seq_len) : count - 1;
    if (all_hi >= count) all_hi = count - 1;
  } else {
    count = a.rows_per_request * a.max_depth;
    all_lo = count;
  }
  if (tid < RT * 16) {
    const int rho = grp * RT * 16 + tid, t = rho / G;
    int lo = 0, hi = count - 1;
    if (anc) {
      lo = t * a.max_depth;
      hi = lo + a.step - 1;
    } else if (extend) {
      lo = within(window_start(seq_len + t, a.window));
      hi = within(seq_len + t);
    }
    if (rho >= R) hi = -1;  // no such row
    sm.loop.seen[tid] = make_int2(lo, hi < count ? hi : count - 1);
  }
  const int ntiles = (count + 31) / 32;

  const uint32_t tp = static_cast<uint32_t>(a.table_page), cpg = static_cast<uint32_t>(a.cache_page);
  const int tp_shift = (tp & (tp - 1)) == 0 ? __builtin_ctz(tp) : -1, cp_shift = (cpg & (cpg - 1)) == 0 ? __builtin_ctz(cpg) : -1;
  char* const sv = sm.loop.v[wave];
  WaveMeta& meta = sm.loop.meta[wave];

  // lane j (and j + 32) looks after key j of a tile: its position (past the split: the last key, which is masked)
  auto key_at = [&](int tile) {
    const int c = tile * 32 + (here(lane) & 31);
    return c < count ? c : count - 1;
  };
  auto lookup = [&](int tile) {
    const int c = key_at(tile);
    if (anc) {  // a column past the row's `step` ancestors takes its first one (masked)
      const int owner = c / here(a.max_depth), dep = c - owner * a.max_depth;
      return a.ancestors[(static_cast<int64_t>(b) * a.rows_per_request + owner) * a.max_depth + (dep < a.step ? dep : 0)];
    }
    const uint32_t pos = static_cast<uint32_t>(start + c), pg = tp_shift >= 0 ? pos >> tp_shift : pos / static_cast<uint32_t>(here(a.table_page));
    return table[pg < static_cast<uint32_t>(x.table_width) ? pg : x.table_width - 1];
  };
  u32x4_t kraw[2][KJ], vraw[NI];
  float ks, vs;
  auto issue = [&](int tile, int32_t ent) {
    uint32_t slot = static_cast<uint32_t>(ent);
    if (!anc) {
      const uint32_t pos = static_cast<uint32_t>(start + key_at(tile));
      slot = slot * tp + (pos - (tp_shift >= 0 ? pos >> tp_shift : pos / static_cast<uint32_t>(here(a.table_page))) * tp);
    }
    uint32_t blk = cp_shift >= 0 ? slot >> cp_shift : slot / static_cast<uint32_t>(here(a.cache_page));
    const uint32_t in = slot - blk * cpg;
    blk = blk < static_cast<uint32_t>(x.num_blocks) ? blk : x.num_blocks - 1;  // (nothing outside the cache is read)
    const int j32 = here(lane) & 31;
    meta.koff[j32] = static_cast<int64_t>(blk) * a.k_stride_page + in * a.k_stride_slot;
    meta.voff[j32] = static_cast<int64_t>(blk) * a.v_stride_page + in * a.v_stride_slot;
    ks = x.k_scale[static_cast<int64_t>(blk) * x.stride_ksb + kvh * x.stride_ksh];
    vs = x.v_scale[static_cast<int64_t>(blk) * x.stride_vsb + kvh * x.stride_vsh];
    const int me = here(lane);
    const char* const kc = static_cast<const char*>(a.keys) + kvh * a.k_stride_head + 16 * (me >> 4);
    const char* const vc = static_cast<const char*>(a.values) + kvh * a.v_stride_head + 16 * (me % CH);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const char* const p = kc + meta.koff[16 * kt + (me & 15)];
#pragma unroll
      for (int j = 0; j < KJ; ++j) kraw[kt][j] = *reinterpret_cast<const u32x4_t*>(p + 64 * j);
      if constexpr (!kEarly) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      // From D = 128 a load of the wave takes whole 128-byte lines of V and needs them no more: with the hint
      // the 64-sequence step takes 130 us in place of 136, a 64-row extend 57 in place of 61. K's lines are read as two
      // halves by two loads, the second half from the cache: the same hint there makes it 143.
      const u32x4_t* const p = reinterpret_cast<const u32x4_t*>(vc + meta.voff[n * RPI + me / CH]);
      vraw[n] = D >= 128 ? __builtin_nontemporal_load(p) : *p;
      if constexpr (!kEarly) __builtin_amdgcn_sched_barrier(0);
    }
  };

  f32x4_t acc[RT][D / 16];
  float m[RT], l[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[r][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const float scale_log2 = a.scale * 1.4426950408889634f;

  // transposing reads of V (Tile8): lane l16 gets d = 16 dt + l16 of keys 16 (k / 4) + 4 g + k % 4, k = l16 / 2
  const auto vread = [](int ln) {
    const int key = 16 * ((ln & 15) >> 3) + 4 * (ln >> 4) + ((ln & 7) >> 1);
    return key * D + 16 * T8::vswz(key) + 8 * (ln & 1);
  };
  // the queries' reads: chunk 8 (c / 2) + 2 g + c % 2 of a row at the chunk xor the row's swizzle (alike for rows 16 apart)
  const auto qread = [](int ln) { return (ln & 15) * 2 * D + 16 * ((2 * (ln >> 4)) ^ Tile<D>::kswz(ln & 15)); };
  if (wave < ntiles) issue(wave, lookup(wave));
  __syncthreads();  // the queries
  int32_t ent = wave + NW < ntiles ? lookup(wave + NW) : 0;
  for (int tile = wave; tile < ntiles; tile += NW) {
    const int base = tile * 32, qnow = qread(here(lane));
    f32x4_t s[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) s[r][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KJ; ++j) {  // steps 2 j and 2 j + 1 take d = 64 j + 16 g + 0 .. 7 and + 8 .. 15
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        u32x4_t q[RT];
        const int qc = qnow ^ 16 * ((8 * j + c) & 15);
#pragma unroll
        for (int r = 0; r < RT; ++r) q[r] = *reinterpret_cast<const u32x4_t*>(sm.loop.q + qc + r * 32 * D + 256 * (j / 2));
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const u32x4_t k16 = __builtin_bit_cast(
              u32x4_t, widen_fp8x8<T>(c ? make_uint2(kraw[kt][j][2], kraw[kt][j][3]) : make_uint2(kraw[kt][j][0], kraw[kt][j][1])));
#pragma unroll
          for (int r = 0; r < RT; ++r) s[r][kt] = mfma16<T>(k16, q[r], s[r][kt]);
        }
        if constexpr (!kEarly) __builtin_amdgcn_sched_barrier(0);
      }
    }
    // a tile that every row sees whole, or not
    const bool full = base >= all_lo && base + 31 <= all_hi;
    const int j32 = here(lane) & 31;
    const bool none = __builtin_fabsf(vs) < 0x1p-100f;
    meta.ks[j32] = ks * scale_log2;
    meta.lv[j32] = none ? 0.f : log2f(vs);
    meta.iv[j32] = none ? 1.f : 1.f / vs;
    if (__any(none)) {  // such a page's values are zeros whatever its codes
      const uint32_t which = static_cast<uint32_t>(__ballot(none));
      const int first = here(lane) / CH;
#pragma unroll
      for (int n = 0; n < NI; ++n)
        if ((which >> (n * RPI + first)) & 1) vraw[n] = u32x4_t{0u, 0u, 0u, 0u};
    }
    auto put_v = [&]() {
      const int me = here(lane);
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int row = n * RPI + me / CH;
        *reinterpret_cast<u32x4_t*>(sv + row * D + 16 * ((me % CH) ^ T8::vswz(row))) = vraw[n];
      }
    };
    put_v();
    auto visible = [&](int2 seen, int k) { return base + k >= seen.x && base + k <= seen.y; };
    if (!full) {
      uint32_t odd = 0;
#pragma unroll
      for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) odd |= nan_bytes(vraw[n][i]);
      if (__any(odd != 0)) {
        for (int k = here(0); k < 32; ++k)
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(sv + k * D + 16 * (dt ^ T8::vswz(k)) + 4 * g);
            const uint32_t bad = nan_bytes(w);
            if (bad == 0) continue;
#pragma unroll
            for (int r = 0; r < RT; ++r)
              if (visible(sm.loop.seen[16 * r + l16], k))
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if ((bad >> (8 * i)) & 0x80u) acc[r][dt][i] = NAN;
          }
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w = here(vraw[n][i]);
            vraw[n][i] = w & ~((nan_bytes(w) >> 7) * 0xffu);
          }
        put_v();
      }
    }
    const auto next = [&]() {
      __builtin_amdgcn_sched_barrier(0);
      if (tile + NW < ntiles) {
        issue(tile + NW, ent);
        if (tile + 2 * NW < ntiles) ent = lookup(tile + 2 * NW);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (kEarly) next();

    u32x4_t pb[RT], pl[kParts == 2 ? RT : 1];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float top = -INFINITY;
      int2 seen = {0, 0};
      if (!full) seen = sm.loop.seen[16 * r + l16];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const f32x4_t k4 = *reinterpret_cast<const f32x4_t*>(&meta.ks[16 * kt + 4 * g]);
        const f32x4_t v4 = *reinterpret_cast<const f32x4_t*>(&meta.lv[16 * kt + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[r][kt][i] = s[r][kt][i] * k4[i] + v4[i];
          if (!full && !visible(seen, 16 * kt + 4 * g + i)) s[r][kt][i] = -INFINITY;
          top = fmaxf(top, s[r][kt][i]);
        }
      }
      if (__any(top > m[r] + kSlack)) {
        float all = fmaxf(top, __shfl_xor(top, 16, 64));
        all = fmaxf(all, __shfl_xor(all, 32, 64));
        const float now = fmaxf(m[r], all);
        const float keep = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - now);
        m[r] = now;
        l[r] *= keep;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[r][i] *= keep;
      }
      const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const f32x4_t i4 = *reinterpret_cast<const f32x4_t*>(&meta.iv[16 * kt + 4 * g]);
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = __builtin_amdgcn_exp2f(s[r][kt][i] - ref);
          l[r] += p[i] == 0.f ? 0.f : p[i] * i4[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t w = pack2<e4::Bf16>(p[2 * i], p[2 * i + 1]);
          pb[r][2 * kt + i] = w;
          if constexpr (kParts == 2)
            pl[r][2 * kt + i] = pack2<e4::Bf16>(p[2 * i] - __uint_as_float(w << 16), p[2 * i + 1] - __uint_as_float(w & 0xffff0000u));
        }
      }
    }
    if constexpr (!kEarly) next();
    const int vnow = vread(here(lane));
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const u32x4_t v16 = __builtin_bit_cast(u32x4_t, widen_fp8x8<e4::Bf16>(lds_tr8(sv + (vnow ^ 16 * (dt & 7)) + 128 * (dt / 8))));
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[r][dt] = mfma16<e4::Bf16>(v16, pb[r], acc[r][dt]);
      if constexpr (kParts == 2)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r][dt] = mfma16<e4::Bf16>(v16, pl[r], acc[r][dt]);
      if constexpr (!kEarly)
        if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }

  // the waves' sums joined: weights 2^(m - the largest m)
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] += __shfl_xor(l[r], 16, 64);
    l[r] += __shfl_xor(l[r], 32, 64);
  }
  __syncthreads();
  if (g == 0) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      sm.join.m[wave][16 * r + l16] = m[r];
      sm.join.l[wave][16 * r + l16] = l[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, sm.join.m[w][16 * r + l16]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = sm.join.m[w][16 * r + l16], lw = sm.join.l[w][16 * r + l16];
      if (mw > -INFINITY || lw != lw) sum += (mw > -INFINITY ? exp2f(mw - top) : 1.f) * lw;
    }
    const float mine = m[r] > -INFINITY ? exp2f(m[r] - top) : 0.f;
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    const int rho = (grp * RT + r) * 16 + here(l16);
    const bool row_in = rho < R;
    const int64_t part = ((static_cast<int64_t>(b) * a.heads + kvh * G + (row_in ? rho % G : 0)) * (a.splits + 1) + split) * a.rows_padded + rho / G;
    if (row_in && wave == 0 && g == 0) a.part_lse[part] = sum != 0.f ? top + log2f(sum) : -INFINITY;
    constexpr int H = Smem<D, RT>::kHalves, C = D / 16 / H;
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int dt = 0; dt < C; ++dt) sm.join.acc[wave][dt][lane] = acc[r][C * h + dt] * (mine * inv);
      __syncthreads();
      if (row_in) {
#pragma unroll
        for (int i = 0; i < C / NW; ++i) {
          const int dt = wave + NW * i;
          f32x4_t o = sm.join.acc[0][dt][lane];
#pragma unroll
          for (int w = 1; w < NW; ++w) o += sm.join.acc[w][dt][lane];
          *reinterpret_cast<f32x4_t*>(a.part_out + part * D + 16 * (C * h + dt) + 4 * g) = o;
        }
      }
      __syncthreads();
    }
  }
}

// The splits of each (row, query head) merged; a row that saw no key gives zeros.
template <int D, int SG, typename T>
__global__ __launch_bounds__(256) void row_merge_fp8_kernel(const eagle4_row_attn_args a, int splits) {
  constexpr int LP = D / 4, PAIRS = 256 / LP / SG;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * PAIRS + threadIdx.x / (LP * SG);
  const int d = 4 * (threadIdx.x % LP);
  const bool ok = pair < static_cast<int64_t>(a.bs) * a.rows_per_request * a.heads;
  const int64_t row = pair / a.heads;
  const int head = static_cast<int>(pair % a.heads);
  const int64_t b = row / a.rows_per_request, t = row % a.rows_per_request;
  const int64_t part0 = ((b * a.heads + head) * (a.splits + 1)) * a.rows_padded + t;
  f32x4_t acc;
  float wsum;
  const bool mine = merge_partials<D, SG>(ok ? splits : 0, [&](int i) { return part0 + static_cast<int64_t>(i) * a.rows_padded; },
                                          a.part_out, a.part_lse, acc, wsum);
  if (!mine || !ok) return;
  const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
  uint16_t* o = static_cast<uint16_t*>(a.out) + row * a.stride_o_row + static_cast<int64_t>(head) * a.stride_o_head + d;
  *reinterpret_cast<uint2*>(o) = make_uint2(T::pack(acc.x * inv, acc.y * inv), T::pack(acc.z * inv, acc.w * inv));
}

// The splits that are used of those that the caller has scratch for: as many as fill the GPU's 256 CUs with resident workgroups
// once, but none of fewer than 256 keys, as far as the window or the page table bound them. A workgroup's start and
// end cost as much as some tiles: 32 requests' extends (54 rows a head, D 256, window 2048) 53 us with 2 splits, 60 with 1, 88 with 8; 64
// draft steps (16 rows, D 128, window 4096) 113 with 2, 112 with 4, 119 with 8, 175 with 1, 171 with 32; one over 4096 keys 39.5 with 1,
// 11.4 with 16, 13.5 with 64.
int used_splits(const eagle4_row_attn_fp8_args& x, int resident, int groups) {
  const eagle4_row_attn_args& a = x.rows;
  const int64_t bound = a.window > 0 ? static_cast<int64_t>(a.window) + a.rows_per_request : static_cast<int64_t>(x.table_width) * a.table_page;
  const int64_t programs = static_cast<int64_t>(a.bs) * a.kv_heads * groups;
  int64_t n = (256 * resident + programs / 2) / programs;
  n = n < (bound + 255) / 256 ? n : (bound + 255) / 256;
  n = n < a.splits ? n : a.splits;
  return n > 1 ? static_cast<int>(n) : 1;
}

template <int D, typename T, int RT>
int launch(const eagle4_row_attn_fp8_args& x, hipStream_t s) {
  const eagle4_row_attn_args& a = x.rows;
  const int R = a.rows_per_request * (a.heads / a.kv_heads);
  const int groups = (R + 16 * RT - 1) / (16 * RT);
  const int splits = used_splits(x, kResident<D, RT>, groups) + (a.step == 0 ? 0 : 1);
  const int64_t grid = (static_cast<int64_t>(splits) * a.kv_heads * a.bs + 7) / 8 * 8 * groups;
  const int64_t pairs = static_cast<int64_t>(a.bs) * a.rows_per_request * a.heads;
  // (both launches have 256 threads a workgroup: under 2^32; the merge takes more than one run a row only in small grids)
  if (grid >= (1 << 24) || (pairs + 1024 / D - 1) / (1024 / D) >= (1 << 24)) return EAGLE4_NOT_COVERED;
  row_attention_fp8_kernel<D, T, RT><<<static_cast<unsigned>(grid), NT, 0, s>>>(x, groups, splits);
  return with_merge_runs<D>(splits, pairs, [&](auto runs) {
    constexpr int SG = decltype(runs)::value;
    constexpr int64_t per = 256 / (D / 4) / SG;
    row_merge_fp8_kernel<D, SG, T><<<static_cast<unsigned>((pairs + per - 1) / per), 256, 0, s>>>(a, splits);
    return E4_LAUNCH_STATUS();
  });
}

template <int D, typename T>
int launch_rows(const eagle4_row_attn_fp8_args& x, hipStream_t s) {
  const int R = x.rows.rows_per_request * (x.rows.heads / x.rows.kv_heads);
  if (R <= 16) return launch<D, T, 1>(x, s);
  if (R <= 32 || D == 256) return launch<D, T, 2>(x, s);
  if constexpr (D < 256) return launch<D, T, 4>(x, s);
}

template <typename T>
int launch_d(const eagle4_row_attn_fp8_args& x, hipStream_t s) {
  switch (x.rows.head_dim) {
    case 64: return launch_rows<64, T>(x, s);
    case 128: return launch_rows<128, T>(x, s);
    case 256: return launch_rows<256, T>(x, s);
    default: return EAGLE4_NOT_COVERED;
  }
}

}  // namespace

extern "C" int eagle4_row_attention_fp8(const eagle4_row_attn_fp8_args* x, void* stream) {
  const eagle4_row_attn_args* a = &x->rows;
  if (a->bs == 0 || a->rows_per_request == 0) return EAGLE4_OK;
  const auto al16 = [](const void* p) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (a->kv_heads <= 0 || a->heads <= 0 || a->heads % a->kv_heads || a->splits < 1 || a->splits > 65535 || a->bs < 0 || a->bs > 65535 ||
      a->step < 0 || a->rows_per_request < 1 || a->rows_padded < a->rows_per_request || a->table == nullptr || a->seq_lens.ptr == nullptr ||
      a->table_page < 1 || a->cache_page < 1 || x->num_blocks < 1 || x->table_width < 1 || x->table_height < 1 ||
      x->k_scale == nullptr || x->v_scale == nullptr || (a->step > 0 && (a->ancestors == nullptr || a->max_depth < a->step)) ||
      (a->dtype != EAGLE4_BF16 && a->dtype != EAGLE4_F16) || !al16(a->q) || !al16(a->keys) || !al16(a->values) || !al16(a->part_out) ||
      a->part_lse == nullptr || a->stride_q_row % 8 || a->stride_q_head % 8 || a->k_stride_page % 16 || a->k_stride_slot % 16 ||
      a->k_stride_head % 16 || a->v_stride_page % 16 || a->v_stride_slot % 16 || a->v_stride_head % 16 || a->out == nullptr ||
      reinterpret_cast<uintptr_t>(a->out) % 8 || a->stride_o_row % 4 || a->stride_o_head % 4 ||
      a->part_rows < static_cast<int64_t>(a->bs) * a->heads * (a->splits + 1) * a->rows_padded)
    return EAGLE4_NOT_COVERED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == EAGLE4_BF16 ? launch_d<e4::Bf16>(*x, s) : launch_d<e4::F16>(*x, s);
}
