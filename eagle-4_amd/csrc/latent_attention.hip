// Tree-verify attention over latent rows on gfx950: every head's key is a token's cached row c of RANK + ROPE values, its
// value the row's first RANK.
//
// Mathematics. For a query row (draft token, head): o = sum_k softmax_k(scale q . c_k) c_k[0..RANK), keys the request's
// context and the round's rows in the draft token's ancestor mask. One pass with a running maximum and sum (log2 domain).
//
// What bounds it. A request's width x heads query rows share every key: 2 (2 RANK + ROPE) operations a row and key against
// 2 (RANK + ROPE) bytes a key (16-bit pages). From about 128 rows on that is the matrix cores' work, below it HBM's.
//
// Split. A workgroup takes ROWS query rows (16, 32 or 64) and a run of 32-key tiles, which all eight waves read from LDS:
//   - RW row waves of 16 rows each; the DW = 8 / RW waves of the same rows share out the output's columns, and the scores
//     between two of them: one takes a tile's keys 0-15, the other 16-31 (with more than two, two sets of them do the
//     same), and they exchange the weights and their running maxima through LDS;
//   - S^T = C Q^T on v_mfma_f32_16x16x32, so that a lane holds scores of one query row and P^T is the B operand of
//     O^T = C^T P^T in the registers' own order; C^T is read by transposing LDS loads of the same tile: a row of the cache
//     is brought in once for both products;
//   - a tile's scores are computed beside the last tile's output, so that the exchange costs no wait: one barrier a tile.
// Scores, maxima, sums and outputs are in 32 bits. The weights alone are rounded to the rows' type, as the matrix cores take them
// (relative to a maximum that moves by whole powers of two): each is off by half a step at most, as the outputs are when they
// are stored, and the two together make the error against 64 bits 0.0023 in bf16 where the outputs' rounding makes 0.0017.
// The launch is one workgroup a CU; each takes an equal run of all (request, row group, tile)s, so requests of any
// lengths fill the chip. A row group cut by a run's end leaves normalised fp32 partials with their log2-sum-exps (at most two
// a workgroup), which a second kernel merges.
//
// Measured (RANK 512, ROPE 64, graph replays). 64 trees of up to 16 tokens, 16 heads, contexts of 1024 to 8192, bf16: 231 us,
// 505 TFLOP/s; four waves that each take all scores of their rows: 455. A tile of 64 rows costs about 3300 cycles, of which
// the products are 1100 and their operands' LDS reads about as much; the rest is the barrier (250 to 650), the exchange of
// weights and the lookups (900 to 1600, with the lookups of each tile on their own instead of four tiles at once: 281 us).
// 128 requests of 4 tokens, 16 heads, fp8 pages: 175 us; widening the codes is a fourth of a tile. 64 single tokens of 16
// heads: 67 us, 4.5 TB/s. One token of 128 heads over 2048 keys: 25.5 us. By stamps in the kernel 15.9 of them lie between the
// first workgroup's start and the last one's end: 1.0 for the counts of tiles, 1.2 to the piece's request, 1.6 for lookups,
// queries and first tiles, 0.7 for the zeroed tile, 1.2 an iteration (16 rows; of 2 to 4), 0.7 for the output, and in runs that
// reach into a second row group the last four again. Launch and drain are some 4, the merge 6. Queries loaded by each lane on its
// own, 16 bytes of every row: 6 us more.

#include "attention_tile.h"

namespace {

using namespace e4attn;

constexpr int kKeys = 32;      // keys of a tile
constexpr int kBatch = 4;      // tiles whose keys' addresses are looked up together
constexpr int kMaxReqs = 512;  // requests of one launch (a thread counts the tiles of each)

struct LatentPlan {
  int first, reqs;       // requests of this launch
  int groups;            // workgroups
  int least;             // tiles of a workgroup's run at least
  int rows;              // query rows of a workgroup at most
  int page_shift;        // of a page size that is a power of two, else -1
  uint32_t page_inv;     // floor(2^32 / page) of any other
  int64_t pre_off, lse_off, part_off;  // float offsets into the workspace
};

constexpr float kNone = -3.0e38f;  // the maximum of no score

// Bytes behind keys that are not there: a position past the context, a page outside the cache.
__device__ __attribute__((aligned(16))) const uint32_t zero_row[640 / 2] = {};

struct Unit {
  int64_t start;          // first token
  int width, context;     // rows, committed positions
  int ctx_tiles, tiles;   // tiles of a row group
  E4_DEV int row_groups(int heads, int rows) const { return (width * heads + rows - 1) / rows; }
};

E4_DEV Unit unit_of(const eagle4_latent_attn_args& a, int b) {
  Unit u;
  u.start = e4::ld(a.query_start_loc, b);
  int64_t width = e4::ld(a.query_start_loc, b + 1) - u.start;
  if (u.start < 0 || width < 0 || u.start + width > a.tokens) width = 0;
  u.width = static_cast<int>(width < a.max_query_len ? width : a.max_query_len);
  int64_t context = e4::ld(a.context_lens, b);
  const int64_t capacity = static_cast<int64_t>(a.max_blocks) * a.page;
  context = context < 0 ? 0 : (context > capacity ? capacity : context);
  u.context = static_cast<int>(context);
  u.ctx_tiles = (u.context + kKeys - 1) / kKeys;
  u.tiles = u.ctx_tiles + (u.width + kKeys - 1) / kKeys;
  return u;
}

E4_DEV uint32_t lds_addr(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p));
}
// 64 lanes x 16 bytes from per-lane addresses into LDS [lds, lds + 1024), lane p at lds + 16 p.
E4_DEV void dma16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
// The same with 4 bytes a lane.
E4_DEV void dma4(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
template <int N>
E4_DEV void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 8 fp8 codes times a power of two, as 16-bit T: exact within split_scale's limits.
template <typename T>
E4_DEV u32x4_t widen8(u32x2_t raw, float pow2) {
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (T::code == EAGLE4_BF16) {
      w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], pow2, false));
      w[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], pow2, true));
    } else {
      w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[i], pow2, false));
      w[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[i], pow2, true));
    }
  }
  return w;
}
// A page's scale as pow2 x rest, 1 <= |rest| < 2: the power goes into the codes as they are widened, the rest (1 for the
// scales that the cache's writer makes) onto the key's score and weight. Neither takes a 16-bit weight out of its range,
// as the whole scale would. The power stays where the largest code (448) and the smallest (2^-9) times it are numbers of T; what
// is beyond joins the rest. (fp16: rows of up to 65504 have scales of up to 2^8, and 256 x 2^8 would be an infinity.)
template <typename T>
E4_DEV void split_scale(float scale, float& pow2, float& rest) {
  constexpr float kLeast = T::code == EAGLE4_BF16 ? 0x1p-117f : 0x1p-15f, kMost = T::code == EAGLE4_BF16 ? 0x1p119f : 0x1p7f;
  const uint32_t e = __float_as_uint(scale) & 0x7f800000u;
  const bool plain = e != 0 && e != 0x7f800000u;
  pow2 = plain ? fminf(fmaxf(__uint_as_float(e), kLeast), kMost) : 1.f;
  rest = plain ? scale / pow2 : scale;
}

// A value that all lanes hold, in scalar registers (what comes from LDS or a table is in vector registers otherwise).
E4_DEV int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
E4_DEV uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
E4_DEV int64_t uniform(int64_t x) {
  return static_cast<int64_t>(static_cast<uint64_t>(uniform(static_cast<uint32_t>(x >> 32))) << 32 |
                              uniform(static_cast<uint32_t>(x)));
}

// x, as a value that the compiler cannot have computed before: what follows from it is computed where it is used, not
// kept in registers over the loop (the 64-row form has none to spare).
E4_DEV int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A tile in LDS: CB blocks of 64 columns, each 32 keys x 128 bytes, the eight 16-byte chunks of a key's 128 bytes at
// chunk ^ swz(key). Both operand reads then run at the LDS's full rate (256 bytes a cycle): the scores' (16 keys; the four
// lane groups at chunks 2 g or 2 g + 1) and the transposing one (8 keys at two adjacent chunks). With the lane groups
// at adjacent chunks instead the scores' reads take twice the cycles. An instruction of direct loads fills 8 keys of a block,
// so a lane's address is its key's row plus a constant a block.
E4_DEV int swz(int key) { return 2 * ((key >> 1) & 3) | ((key >> 3) & 1); }

constexpr int kWaves = 8, kThreads = 64 * kWaves;

template <int RANK_, int ROPE, typename T_, bool FP8_, int RW_>
struct Shape {
  using T = T_;
  static constexpr bool FP8 = FP8_;
  static constexpr int RANK = RANK_, RW = RW_, DW = kWaves / RW, DT = RANK / 16 / DW;
  static constexpr int DIM = RANK + ROPE, CB = DIM / 64, KC = DIM / 32, ROWS = RW * 16, TILE = CB * 4096;
  // 16-bit pages: a ring of four tiles, two in use and two on their way. fp8 pages: a ring of three, two in use and one being
  // widened, and one of two tiles of codes, the one that is widened and one on its way.
  static constexpr int NBUF = FP8 ? 3 : 4, RAW = CB * 2048;
  // blocks of 64 columns that waves 0-3 (each 8 keys of a tile) bring in; waves 4-7 bring in the rest
  static constexpr int CB0 = (CB + 1) / 2, CB1 = CB - CB0;
  // LDS operands of the matrix products in registers at a time, the one in use among them. Their loads run that far ahead
  // in this order, product by product: left to itself the compiler waits for each operand right after its load.
  static constexpr int AHEAD = 8;
};

// The larger of a lane's value and that of lane ^ 16 or lane ^ 32: swaps of rows of lanes, no LDS trip.
template <int N>
E4_DEV float other_max(float x) {
  const uint32_t w = __float_as_uint(x);
  const auto r = N == 16 ? __builtin_amdgcn_permlane16_swap(w, w, false, false) : __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A wave's share of the weights: P^T of one half tile (16 keys x 16 rows) as written by its lanes, and the rows' maxima.
template <int RW>
struct Weights {
  __attribute__((aligned(16))) u32x2_t p[RW][2][64];
  float m[RW][2][16];
};

// The scores of keys 16 kt .. of a tile, for a wave's 16 rows. between(c) follows product c: other work, which the matrix
// core's time covers.
template <typename S, typename F>
E4_DEV f32x4_t score_step(const char* tile, const u32x4_t (&q)[S::KC], int kt, int lane, F between) {
  using T = typename S::T;
  const int g = lane >> 4, l16 = lane & 15, x = swz(l16);
  const char* const k0 = tile + kt * 2048 + l16 * 128 + 16 * ((2 * g) ^ x);
  const char* const k1 = tile + kt * 2048 + l16 * 128 + 16 * ((2 * g + 1) ^ x);
  u32x4_t ka[S::AHEAD];
  const auto load = [&](int c) {
    ka[c % S::AHEAD] = *reinterpret_cast<const u32x4_t*>((c & 1 ? k1 : k0) + (c / 2) * 4096);
  };
#pragma unroll
  for (int c = 0; c < S::AHEAD - 1; ++c) load(c);
  f32x4_t s[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};  // two chains: a product waits for the last but one
#pragma unroll
  for (int c = 0; c < S::KC; ++c) {
    if (c + S::AHEAD - 1 < S::KC) load(c + S::AHEAD - 1);
    s[c % 2] = mfma16<T>(ka[c % S::AHEAD], q[c], s[c % 2]);
    between(c);
    __builtin_amdgcn_sched_barrier(0);
  }
  return s[0] + s[1];
}

// The weights of those scores into `to`, relative to the rows' maximum m; l takes their sum. Bit k of bits: key k of the tile
// is visible to the lane's row. In kPhases phases without a branch, for the places between the products of the output.
template <typename S, typename W>
struct WeightStep {
  using T = typename S::T;
  static constexpr int kPhases = 8;
  f32x4_t s, ks;
  float top, p[4];
  E4_DEV void phase(int i, W& to, int row_wave, int kt, bool writes, float& m, float& l, float scale_log2,
                    const float* key_scale, int lane, uint32_t bits) {
    const int g = lane >> 4;
    if (i == 0) {
      s *= scale_log2;
      if constexpr (S::FP8) {
        ks = *reinterpret_cast<const f32x4_t*>(key_scale + 16 * kt + 4 * g);
        s *= ks;
      }
    } else if (i == 1) {
      const uint32_t mine = bits >> (16 * kt + 4 * g);
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = (mine >> k) & 1 ? s[k] : -INFINITY;
    } else if (i == 2) {
      top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
      top = other_max<16>(top);
    } else if (i == 3) {
      top = other_max<32>(top);
    } else if (i == 4) {
      // The maximum moves only when it grows by more than 2^8 (until then p stays below 2^8, which 16 bits hold as well as
      // values below 1), and to a whole number: what was weighted with the last one is then scaled without rounding.
      const float now = top > m + 8.f ? ceilf(top) : m;
      l *= __builtin_amdgcn_exp2f(m - now);
      m = now;
    } else if (i == 5) {
#pragma unroll
      for (int k = 0; k < 4; ++k) p[k] = __builtin_amdgcn_exp2f(s[k] - m);
    } else if (i == 6) {
      l += (p[0] + p[1]) + (p[2] + p[3]);
      if constexpr (S::FP8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] *= ks[k];
      }
    } else if (writes) {
      to.p[row_wave][kt][lane] = u32x2_t{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3])};
      if (g == 0) to.m[row_wave][kt][lane & 15] = m;
    }
  }
};

// Two packed weights times a power of two.
template <typename T>
E4_DEV uint32_t scale2(uint32_t w, float f) {
  return pack2<T>(T::to_f32(static_cast<uint16_t>(w & 0xffffu)) * f, T::to_f32(static_cast<uint16_t>(w >> 16)) * f);
}

// The weights of a tile as the operand of its output. macc is what acc is relative to, m what the wave's own next weights
// are: both move to the largest maximum that the tile's weights bring. (In front of the scores, where no operand of a product
// is in registers: the compiler then keeps one copy of acc over the branch.)
template <typename S, typename W>
E4_DEV u32x4_t take_weights(const W& from, int row_wave, f32x4_t (&acc)[S::DT], float& macc, float& m, float& l,
                            int lane) {
  using T = typename S::T;
  const int l16 = lane & 15;
  // element i of P^T's operand is key 16 (i / 4) + 4 g + i % 4
  u32x2_t p0 = from.p[row_wave][0][lane], p1 = from.p[row_wave][1][lane];
  const float m0 = from.m[row_wave][0][l16], m1 = from.m[row_wave][1][l16];
  if (__any(m0 != macc || m1 != macc)) {
    const float now = fmaxf(macc, fmaxf(m0, m1));
    const float keep = exp2f(macc - now), f0 = exp2f(m0 - now), f1 = exp2f(m1 - now);
    l *= exp2f(m - now);  // m <= now: the wave's own maximum is m0 or m1, or that of waves that do the same
    macc = m = now;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      p0[i] = scale2<T>(p0[i], f0);
      p1[i] = scale2<T>(p1[i], f1);
    }
#pragma unroll
    for (int dt = 0; dt < S::DT; ++dt) acc[dt] *= keep;
  }
  return u32x4_t{p0[0], p0[1], p1[0], p1[1]};
}

// O^T += C^T P^T of a tile, for a wave's 16 rows and its columns dbase ...; between(dt) follows product dt.
template <typename S, typename F>
E4_DEV void value_step(const char* tile, u32x4_t pb, f32x4_t (&acc)[S::DT], int dbase, int lane, F between) {
  using T = typename S::T;
  const int g = lane >> 4, l16 = lane & 15;
  const int j = l16 >> 2, s4 = l16 & 3, kv = 4 * g + j, xv = swz(kv);
  // columns dbase + 16 dt ..: block dbase / 64 + dt / 4, chunks 2 (dt % 4) and the next (waves with fewer than four such
  // tiles share a block: their first is its tile dt0)
  const char* const vrow = tile + kv * 128 + 8 * (s4 & 1) + (dbase / 64) * 4096;
  const int dt0 = dbase % 64 / 16;
  constexpr int VA = S::AHEAD < S::DT ? S::AHEAD : S::DT;
  u32x4_t va[VA];
  const auto load = [&](int dt) {
    const char* const at = vrow + (dt / 4) * 4096 + 16 * ((2 * (dt0 + (dt & 3)) + (s4 >> 1)) ^ xv);
    const v4i16 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(at));
    const v4i16 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(at + 2048));
    const u32x2_t lo = __builtin_bit_cast(u32x2_t, lo4), hi = __builtin_bit_cast(u32x2_t, hi4);
    va[dt % VA] = u32x4_t{lo[0], lo[1], hi[0], hi[1]};
  };
#pragma unroll
  for (int dt = 0; dt < VA - 1; ++dt) load(dt);
#pragma unroll
  for (int dt = 0; dt < S::DT; ++dt) {
    if (dt + VA - 1 < S::DT) load(dt + VA - 1);
    acc[dt] = mfma16<T>(va[dt % VA], pb, acc[dt]);
    between(dt);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// What a workgroup keeps in LDS, for S the shape of the most rows that it may take.
template <typename S>
struct Lds {
  // (sizes are of every shape with these columns and pages, but those of the weights and sums)
  static constexpr int kBatchKeys = kBatch * kKeys, kRowWaves = S::RW;
  __attribute__((aligned(1024))) char smem[S::NBUF][S::TILE];
  __attribute__((aligned(1024))) char s_raw[S::FP8 ? 2 : 1][S::FP8 ? S::RAW : 16];
  Weights<S::RW> s_w[2];
  // The keys of two batches of tiles: their table entries and scales as loaded, then the addresses of their rows, a bit a key
  // that is there, and the two parts of its scale.
  __attribute__((aligned(16))) int32_t s_ent[kBatchKeys];
  __attribute__((aligned(16))) float s_entscale[S::FP8 ? kBatchKeys : 1];
  uint64_t s_row[2][kBatchKeys];
  uint32_t s_vis[2][kBatch];
  __attribute__((aligned(16))) float s_rest[S::FP8 ? 2 : 1][kBatchKeys], s_pow2[S::FP8 ? 2 : 1][kBatchKeys];
  uint32_t s_bad;  // a bit a new key: it holds a value that is not finite
  uint32_t s_tot[2][kWaves];
  float s_sum[S::RW][2][16];
  int s_at;
  uint32_t s_before;
};

// The workgroup's run, S::ROWS rows at a time: `total` tiles in all, `sum_tiles` of the requests up to the thread's and `mine`
// of that one.
template <typename S, typename L>
E4_DEV void latent_rows(const eagle4_latent_attn_args& a, const LatentPlan& p, L& lds, uint32_t total, uint32_t sum_tiles,
                        uint32_t mine) {
  using T = typename S::T;
  constexpr bool FP8 = S::FP8;
  constexpr int RW = S::RW, RANK = S::RANK, kBatchKeys = L::kBatchKeys;
  auto& smem = lds.smem;
  auto& s_raw = lds.s_raw;
  auto& s_w = lds.s_w;
  auto& s_ent = lds.s_ent;
  auto& s_entscale = lds.s_entscale;
  auto& s_row = lds.s_row;
  auto& s_vis = lds.s_vis;
  auto& s_rest = lds.s_rest;
  auto& s_pow2 = lds.s_pow2;
  auto& s_bad = lds.s_bad;
  auto& s_sum = lds.s_sum;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15;
  uint32_t share = (total + p.groups - 1) / p.groups;
  share = share < static_cast<uint32_t>(p.least) ? p.least : share;
  // adjacent runs on one XCD (workgroups go to the eight in turn): row groups of a request share its tiles in the L2
  const int wg = p.groups % 8 == 0 ? (blockIdx.x % 8) * (p.groups / 8) + blockIdx.x / 8 : blockIdx.x;
  uint32_t pos = wg * share;
  const uint32_t stop = pos + share < total ? pos + share : total;
  if (sum_tiles - mine <= pos && pos < sum_tiles) {  // the request of tile `pos`
    lds.s_at = tid;
    lds.s_before = sum_tiles - mine;
  }
  if (wg == 0 && tid < p.reqs) {  // for the merge
    uint32_t* const pre = reinterpret_cast<uint32_t*>(a.workspace + p.pre_off);
    pre[tid + 1] = sum_tiles;
    if (tid == 0) {
      pre[0] = 0;
      pre[p.reqs + 1] = S::ROWS;
    }
  }
  __syncthreads();
  if (pos >= stop) return;
  int at = uniform(lds.s_at);
  uint32_t before = uniform(lds.s_before);  // tiles before request `at`

  const int row_wave = wave / S::DW, column_wave = wave % S::DW, kt = column_wave % 2, dbase = column_wave * S::DT * 16;
  const float scale_log2 = a.scale * 1.4426950408889634f;
  constexpr int EB = FP8 ? 1 : 2;
  const char* const cache = static_cast<const char*>(a.cache);
  const int64_t scb = a.stride_cb * EB, scs = a.stride_cs * EB;
  const auto page_of = [&](int pos) {  // pos / page: by the inverse it comes out right or one short
    if (p.page_shift >= 0) return pos >> p.page_shift;
    const int n = static_cast<int>(__umulhi(static_cast<uint32_t>(pos), p.page_inv));
    return n + (pos - n * a.page >= a.page ? 1 : 0);
  };
  // a wave brings in 8 keys of a tile, 8 lanes a key, half the blocks of columns
  const int octet = wave % 4;
  const bool second_half = wave >= 4;
  const int cb_first = second_half ? S::CB0 : 0;

  while (pos < stop) {
    const int b = p.first + at;
    Unit u = unit_of(a, b);
    u = Unit{uniform(u.start), uniform(u.width), uniform(u.context), uniform(u.ctx_tiles), uniform(u.tiles)};
    const uint32_t within = pos - before;
    const uint32_t its_tiles = static_cast<uint32_t>(u.tiles) * static_cast<uint32_t>(uniform(u.row_groups(a.heads, S::ROWS)));
    if (within >= its_tiles) {
      before += its_tiles;
      ++at;
      continue;
    }
    const int rg = static_cast<int>(within / u.tiles), t0 = static_cast<int>(within % u.tiles);
    const int t1 = static_cast<int>(static_cast<uint32_t>(u.tiles - t0) < stop - pos ? u.tiles : t0 + (stop - pos));
    const int32_t* const table = static_cast<const int32_t*>(a.block_table.ptr) + b * a.block_table.s0;

    const int row0 = rg * S::ROWS + row_wave * 16;
    const bool computes = row0 < u.width * a.heads;
    // the lane's row: its place among the request's rows, its draft token and head (0, 0 for none)
    const auto my_row = [&](int& rho, int& t, int& head) {
      rho = row0 + (fresh(lane) & 15);
      const bool ok = rho < u.width * a.heads;
      t = ok ? rho / a.heads : 0;
      head = ok ? rho - t * a.heads : 0;
      return ok;
    };
    const int tiles = t1 - t0;
    const auto is_ctx = [&](uint32_t i) { return t0 + static_cast<int>(i) < u.ctx_tiles; };  // tile i of the piece
    // The keys of batch n of the piece (tiles kBatch n ..), one a thread of waves 0 and 1: the table entry of a context key
    // (a key behind the context: the last one's), ...
    const auto entry_of = [&](int n, int i) -> const int32_t* {
      const int k = (t0 + kBatch * n) * kKeys + i;
      return table + page_of(k < u.context ? k : (u.context > 0 ? u.context - 1 : 0));
    };
    // ... and from it the key's address, its mark and its scale. What is not there reads zeros.
    const auto fill = [&](int n, int i, int32_t blk, float scale) {
      const int tile = kBatch * n + i / kKeys, key = i % kKeys;
      const char* row = nullptr;
      if (tile < tiles && is_ctx(tile)) {
        const int k = (t0 + tile) * kKeys + key, page = page_of(k);
        if (k < u.context && blk >= 0 && blk < a.num_blocks)
          row = cache + blk * scb + static_cast<int64_t>(k - page * a.page) * scs;
      } else if (tile < tiles) {
        const int j = (t0 + tile - u.ctx_tiles) * kKeys + key;
        scale = 1.f;
        if (j < u.width) row = static_cast<const char*>(a.latent_new) + (u.start + j) * a.stride_nt * 2;
      }
      if (row == nullptr) scale = 1.f;
      const uint64_t there = __ballot(row != nullptr);
      if (key == 0) s_vis[n % 2][i / kKeys] = static_cast<uint32_t>(there >> (i & 32));
      s_row[n % 2][i] = reinterpret_cast<uint64_t>(row != nullptr ? row : reinterpret_cast<const char*>(zero_row));
      if constexpr (FP8) split_scale<T>(scale, s_pow2[n % 2][i], s_rest[n % 2][i]);
    };
    // In the loop the lookups are direct loads too, two iterations ahead of the fill, which is two ahead of the first use.
    const auto lookup = [&](int i) {
      if (wave >= 2) return;
      const int n = i / kBatch, key = fresh(tid), k0 = 64 * wave;
      if (i % kBatch == 2) {
        if ((t0 + kBatch * (n + 2)) * kKeys < u.context) dma4(entry_of(n + 2, key), uniform(lds_addr(&s_ent[k0])));
      } else if (FP8 && i % kBatch == 3) {  // (an entry that was not loaded is none of a key's: in bounds, or taken for none)
        const int32_t blk = s_ent[key];
        const void* const none = zero_row;  // not page 0's scale: a cache of no pages has none
        dma4(blk >= 0 && blk < a.num_blocks ? a.scale_page + blk * a.stride_sp : none,
             uniform(lds_addr(&s_entscale[FP8 ? k0 : 0])));
      } else if (i % kBatch == 0 && i > 0) {
        fill(n + 1, key, s_ent[key], FP8 ? s_entscale[FP8 ? key : 0] : 1.f);
      }
    };
    // Direct loads of a tile, in two parts: the address, then the loads one by one. A tile past the piece (and, for fp8, one
    // of the round's rows) brings in zeros, so that every iteration has the same loads.
    struct Loads {
      const char* src;
      uint32_t dst;
    };
    const auto row_of = [&](int i) {  // of the lane's key of tile i
      const int ln = fresh(lane), key = FP8 ? 16 * (wave % 2) + (ln >> 2) : 8 * octet + (ln >> 3);
      return s_row[i / kBatch % 2][i % kBatch * kKeys + key];
    };
    // 16-bit rows: block c of the wave's CB0 (waves 4-7: CB1) blocks
    const auto prepare = [&](int i, uint64_t at) {
      const int ln = fresh(lane), key = 8 * octet + (ln >> 3), chunk = (ln & 7) ^ swz(key);
      const char* const row = reinterpret_cast<const char*>(at);
      return Loads{row + (16 * chunk + 128 * cb_first),
                   uniform(lds_addr(smem[i % S::NBUF]) + 1024 * octet + 4096 * cb_first)};
    };
    const auto load = [&](const Loads& to, int c) { dma16(to.src + 128 * c, to.dst + 4096 * c); };
    // fp8 codes: a block of 64 columns is 32 keys x 64 bytes, an instruction 16 keys of it; wave w brings in keys 16 (w % 2) ..
    // of blocks w / 2, w / 2 + 4, ..
    const auto prepare8 = [&](int i, uint64_t at) {
      const int ln = fresh(lane);
      const char* row = reinterpret_cast<const char*>(at);
      if (!is_ctx(i)) row = reinterpret_cast<const char*>(zero_row);
      return Loads{row + (16 * (ln & 3) + 64 * (wave / 2)),
                   uniform(lds_addr(s_raw[FP8 ? i % 2 : 0]) + 1024 * (wave % 2) + 2048 * (wave / 2))};
    };
    const auto load8 = [&](const Loads& to, int c) { dma16(to.src + 256 * c, to.dst + 8192 * c); };
    // the loads that every wave has, and the ones that some have beyond them
    constexpr int kLoads = FP8 ? S::CB / 4 : S::CB1;
    const bool more = FP8 ? wave / 2 + 4 * kLoads < S::CB : S::CB0 > S::CB1 && !second_half;
    const auto prepare_next = [&](int i, uint64_t at) {
      if constexpr (FP8) return prepare8(i, at); else return prepare(i, at);
    };
    const auto load_next = [&](const Loads& to, int c) {
      if constexpr (FP8) load8(to, c); else load(to, c);
    };
    const auto load_all = [&](const Loads& to) {
#pragma unroll
      for (int c = 0; c < kLoads; ++c) load_next(to, c);
      if (more) load_next(to, kLoads);
    };
    // widens the codes of block c of the wave's CB0 / CB1 blocks
    struct Codes {
      const char* src;
      char* dst;
      float pow2;
    };
    const auto codes_of = [&](int i) {
      const int ln = fresh(lane), key = 8 * octet + (ln >> 3), chunk = (ln & 7) ^ swz(key);
      return Codes{s_raw[FP8 ? i % 2 : 0] + 2048 * cb_first + key * 64 + 8 * (ln & 7),
                   smem[i % S::NBUF] + 4096 * cb_first + key * 128 + 16 * chunk,
                   s_pow2[FP8 ? i / kBatch % 2 : 0][i % kBatch * kKeys + key]};
    };
    const auto widen = [&](const Codes& x, int c) {
      *reinterpret_cast<u32x4_t*>(x.dst + 4096 * c) = widen8<T>(*reinterpret_cast<const u32x2_t*>(x.src + 2048 * c), x.pow2);
    };
    // fp8, what a tile needs of every wave an iteration ahead: its codes widened, or (the round's rows are 16-bit, and few)
    // its rows brought in
    const auto next_rows = [&](int i) {
      if (i >= tiles) return;
      if (is_ctx(i)) {
        const Codes x = codes_of(i);
#pragma unroll
        for (int c = 0; c < S::CB1; ++c) widen(x, c);
        if (S::CB0 > S::CB1 && !second_half) widen(x, S::CB1);
      } else {
        const int key = 8 * octet + (fresh(lane) >> 3);
        const Loads to = prepare(i, s_row[i / kBatch % 2][i % kBatch * kKeys + key]);
#pragma unroll
        for (int c = 0; c < S::CB1; ++c) load(to, c);
        if (S::CB0 > S::CB1 && !second_half) load(to, S::CB1);
      }
    };

    __syncthreads();  // the last piece's tiles have been read
    // The queries come in through the last two tiles' place, whole lines once for all waves: a lane's own loads would be 16
    // bytes of every row, twice. 8 rows x 64 columns an instruction, in the layout of a tile. Waves 4-7 have these loads, as
    // waves 0-3 have the lookups, whose waits would take them in.
    char* const s_q = smem[S::NBUF - 2];
    static_assert(S::KC / 2 * S::ROWS * 128 <= 2 * S::TILE, "the queries' place");
    if (second_half) {
#pragma unroll 1
      for (int part = wave - 4; part < 2 * RW; part += 4) {
        const int ln = fresh(lane), row = 8 * part + (ln >> 3), rho = rg * S::ROWS + row;
        const bool ok = rho < u.width * a.heads;
        const int t = ok ? rho / a.heads : 0, head = ok ? rho - t * a.heads : 0;
        const char* const src = ok ? reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.q) +
                                                                   (u.start + t) * a.stride_qt + head * a.stride_qh)
                                   : reinterpret_cast<const char*>(zero_row);
        const int chunk = 16 * ((ln & 7) ^ swz(row % kKeys));
        const uint32_t dst = uniform(lds_addr(s_q) + 1024 * part);
#pragma unroll 1
        for (int cb = 0; cb < S::KC / 2; ++cb) dma16(src + 128 * cb + chunk, dst + cb * S::ROWS * 128);
      }
    }
    if (tid < 2 * kBatchKeys) {  // batches 0 and 1
      const int n = tid / kBatchKeys, i = tid % kBatchKeys;
      int32_t blk = -1;
      if ((t0 + kBatch * n) * kKeys + i < u.context) blk = *entry_of(n, i);
      float scale = 1.f;
      if (FP8 && blk >= 0 && blk < a.num_blocks) scale = a.scale_page[blk * a.stride_sp];
      fill(n, i, blk, scale);
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < 2; ++i) load_all(prepare_next(i, row_of(i)));
    if constexpr (FP8) {
      wait_vm<0>();
      __syncthreads();
      next_rows(0);
    } else {  // the queries are there; the two tiles may be on their way
      if (second_half) wait_vm<2 * S::CB1>();
      __syncthreads();
    }
    // Waits until tile i (fp8: the codes of the one after it too) is there for every wave, the last tile's weights too; the
    // buffer of the tile before that is free.
    const auto arrive = [&](int i) {
      if (FP8 || i == tiles) {
        wait_vm<0>();
      } else {  // the loads of the tile behind it may be outstanding
        if (second_half) wait_vm<S::CB1>(); else wait_vm<S::CB0>();
      }
      __syncthreads();
    };
    // The round's rows. One that is not finite must not reach the rows that do not see it through 0 x NaN: it is cleared, and
    // the rows that see it become NaN. Gives a bit a row that was cleared; every wave calls it.
    const auto clean = [&](int i) {
      if (tid == 0) s_bad = 0;
      __syncthreads();
      const int ln = fresh(lane), my_key = 8 * octet + (ln >> 3);
      char* const mine = smem[i % S::NBUF] + 4096 * cb_first + my_key * 128 + 16 * (ln & 7);
      bool bad = false;
#pragma unroll 1
      for (int c = 0; c < (second_half ? S::CB1 : S::CB0); ++c) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(mine + 4096 * c);
        constexpr uint32_t kExp = T::code == EAGLE4_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
        for (int k = 0; k < 4; ++k) bad |= (w[k] & kExp) == kExp || ((w[k] >> 16) & kExp) == kExp;
      }
      if (bad) atomicOr(&s_bad, 1u << my_key);
      __syncthreads();
      const uint32_t poison = __builtin_amdgcn_readfirstlane(s_bad);
      if (poison != 0) {
        if ((poison >> my_key) & 1) {
#pragma unroll 1
          for (int c = 0; c < (second_half ? S::CB1 : S::CB0); ++c)
            *reinterpret_cast<u32x4_t*>(mine + 4096 * c) = u32x4_t{0u, 0u, 0u, 0u};
        }
        __syncthreads();
      }
      return poison;
    };
    u32x4_t q[S::KC];
    {
      const int ln = fresh(lane), row = 16 * row_wave + (ln & 15);
      const char* const from = s_q + row * 128;
#pragma unroll
      for (int c = 0; c < S::KC; ++c)  // the columns of the lane's chunk of the scores' operand
        q[c] = *reinterpret_cast<const u32x4_t*>(from + c / 2 * (S::ROWS * 128) +
                                                 16 * ((2 * (ln >> 4) + (c & 1)) ^ swz(row % kKeys)));
      // Settled here, once: a wait for them inside the loop would wait for the tiles on their way too.
#pragma unroll
      for (int c = 0; c < S::KC; ++c) asm volatile("" : "+v"(q[c]));
    }
    __syncthreads();
    // The first iteration's output: no weights over a tile of zeros.
    for (int i = tid; i < S::TILE / 16; i += kThreads)
      *reinterpret_cast<u32x4_t*>(smem[S::NBUF - 1] + 16 * i) = u32x4_t{0u, 0u, 0u, 0u};
    if (tid < RW * 64) {
      s_w[1].p[tid / 64][0][lane] = s_w[1].p[tid / 64][1][lane] = u32x2_t{0u, 0u};
      if (lane < 32) s_w[1].m[tid / 64][lane / 16][l16] = kNone;
    }
    if (!computes) {  // no rows of this row group: a share of the loads alone
      for (int i = 0; i <= tiles; ++i) {
        arrive(i);
        if (i == tiles) break;
        lookup(i);
        const Loads to = prepare_next(i + 2, row_of(i + 2));
        if (!is_ctx(i)) clean(i);
        load_all(to);
        if constexpr (FP8) next_rows(i + 1);
      }
      __syncthreads();
      pos += tiles;
      continue;
    }
    f32x4_t acc[S::DT];
    float m = kNone, macc = kNone, l = 0.f;
#pragma unroll
    for (int dt = 0; dt < S::DT; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // Iteration i: the scores of tile i, beside them the loads of the tile two ahead; the output of the tile before it, beside
    // that the scores' weights.
    for (int i = 0; i <= tiles; ++i) {
      arrive(i);
      const u32x4_t pb = take_weights<S>(s_w[(i + 1) % 2], row_wave, acc, macc, m, l, fresh(lane));
      using Step = WeightStep<S, Weights<L::kRowWaves>>;
      Step w;
      w.s = f32x4_t{0.f, 0.f, 0.f, 0.f};
      uint32_t bits = 0;
      if (i < tiles) {
        const uint64_t next_row = row_of(i + 2);
        bits = s_vis[i / kBatch % 2][i % kBatch];
        const Loads to = prepare_next(i + 2, next_row);
        if (!is_ctx(i)) {
          const uint32_t poison = clean(i);
          int rho, t, head;
          const uint64_t mask = my_row(rho, t, head) ? static_cast<uint64_t>(a.masks[b * a.stride_mask + t]) : 0;
          bits &= static_cast<uint32_t>(mask >> ((t0 + i - u.ctx_tiles) * kKeys));
          if (bits & poison) l = __builtin_nanf("");
        }
        w.s = score_step<S>(smem[i % S::NBUF], q, kt, fresh(lane), [&](int c) {
          if (c % 2 == 1 && c / 2 < kLoads) load_next(to, c / 2);
        });
        if (more) load_next(to, kLoads);
        lookup(i);
        if constexpr (FP8) next_rows(i + 1);
      }
      const int ln = fresh(lane);
      const float* const rest = s_rest[FP8 ? i / kBatch % 2 : 0] + i % kBatch * kKeys;
      value_step<S>(smem[(i + S::NBUF - 1) % S::NBUF], pb, acc, dbase, ln, [&](int dt) {
        constexpr int kPhases = Step::kPhases;
#pragma unroll
        for (int ph = 0; ph < kPhases; ++ph)
          if (ph * S::DT / kPhases == dt)
            w.phase(ph, s_w[i % 2], row_wave, kt, column_wave < 2, m, l, scale_log2, rest, ln, bits);
      });
    }
    // the sum over both halves of the keys: each wave's own is relative to the last maximum by now
    const int ln = fresh(lane), g = ln >> 4, l16 = ln & 15;
    float sum = l + __shfl_xor(l, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (column_wave < 2 && g == 0) s_sum[row_wave][kt][l16] = sum;
    __syncthreads();
    sum = s_sum[row_wave][0][l16] + s_sum[row_wave][1][l16];

    const bool whole = t0 == 0 && t1 == u.tiles;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // nothing seen: zeros
    int rho, t, head;
    const bool ok = my_row(rho, t, head);
    if (whole) {
      uint16_t* const o = static_cast<uint16_t*>(a.out) + (u.start + t) * a.stride_ot + head * a.stride_oh + dbase;
      // Two column tiles at a time: rows of lanes swapped, a lane has 8 adjacent columns of one of them (16 bytes a store).
#pragma unroll
      for (int dt = 0; dt < S::DT; dt += 2) {
        uint32_t w[2][2];  // [half of a lane's columns][word]
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const auto r = __builtin_amdgcn_permlane16_swap(pack2<T>(acc[dt][2 * k] * inv, acc[dt][2 * k + 1] * inv),
                                                          pack2<T>(acc[dt + 1][2 * k] * inv, acc[dt + 1][2 * k + 1] * inv),
                                                          false, false);
          w[0][k] = r[0];
          w[1][k] = r[1];
        }
        if (ok) *reinterpret_cast<u32x4_t*>(o + 16 * (dt + (g & 1)) + 8 * (g >> 1)) = u32x4_t{w[0][0], w[0][1], w[1][0], w[1][1]};
      }
    } else if (ok) {
      const int64_t part = (2 * static_cast<int64_t>(wg) + (t0 == 0 ? 1 : 0)) * S::ROWS + rho - rg * S::ROWS;
      float* const o = a.workspace + p.part_off + part * RANK + dbase;
#pragma unroll
      for (int dt = 0; dt < S::DT; ++dt) *reinterpret_cast<f32x4_t*>(o + 16 * dt + 4 * g) = acc[dt] * inv;
      if (g == 0 && dbase == 0) a.workspace[p.lse_off + part] = sum == 0.f ? -INFINITY : macc + log2f(sum);
    }
    pos += tiles;
  }
}

// Tiles of 64 rows up to which a launch takes 16 rows a workgroup: 2.5 a workgroup. 64 rows share a tile's loads best, but where
// there is so little work 16 spread it over more workgroups, with less to bring in, to leave and to merge (RANK 512; the times
// with 64 and 16 rows: one token of 128 heads over 2048 keys, 130 tiles: 34.5 and 25.4 us; 8192 keys, 514: 45.4 and 34.1;
// 16384 keys, 1026: 52.2 and 46.2; 32768 keys, 2050: 60.8 and 66.4; a tree of 16 x 16 heads over 4096 keys, 516: 34.0 and
// 31.3; 4 such trees over 512 keys, 272: 36.3 and 27.0; over 2048 keys, 1040: 34.1 and 40.6). The contexts decide, not the
// tables' width, which in an engine is that of its longest context: chosen on the GPU, in one kernel that holds both forms.
constexpr uint32_t kFewTiles = 640;

// Of 16 (FORM 1) or 32 rows (2) a workgroup, or (4) of 64 or 16, by the tiles that there are.
template <int RANK, int ROPE, typename T, bool FP8, int FORM>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void latent_kernel(
    const eagle4_latent_attn_args a, const LatentPlan p) {
  using S = Shape<RANK, ROPE, T, FP8, FORM>;
  __shared__ Lds<S> lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // tiles before each request (one a thread), and the same of 16 rows
  static_assert(kMaxReqs <= kThreads, "requests of a launch");
  uint32_t mine = 0, few = 0;
  if (tid < p.reqs) {
    const Unit u = unit_of(a, p.first + tid);
    mine = static_cast<uint32_t>(u.tiles) * static_cast<uint32_t>(u.row_groups(a.heads, S::ROWS));
    if constexpr (FORM == 4) few = static_cast<uint32_t>(u.tiles) * static_cast<uint32_t>(u.row_groups(a.heads, 16));
  }
  uint32_t sum = mine, sum_few = few;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const uint32_t o = __shfl_up(sum, k, 64);
    if (lane >= k) sum += o;
    if constexpr (FORM == 4) {
      const uint32_t f = __shfl_up(sum_few, k, 64);
      if (lane >= k) sum_few += f;
    }
  }
  if (lane == 63) {
    lds.s_tot[0][wave] = sum;
    lds.s_tot[1][wave] = sum_few;
  }
  __syncthreads();
  uint32_t total = 0, total_few = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) sum += lds.s_tot[0][w];
    total += lds.s_tot[0][w];
    if constexpr (FORM == 4) {
      if (w < wave) sum_few += lds.s_tot[1][w];
      total_few += lds.s_tot[1][w];
    }
  }
  total = uniform(total);
  if constexpr (FORM == 4) {
    if (total <= kFewTiles) {
      latent_rows<Shape<RANK, ROPE, T, FP8, 1>>(a, p, lds, uniform(total_few), sum_few, few);
      return;
    }
  }
  latent_rows<S>(a, p, lds, total, sum, mine);
}

// Rows of row groups that were cut: their partials by log2-sum-exp, a thread four columns: 1024 / RANK rows a workgroup.
template <int RANK, typename T>
__global__ __launch_bounds__(256) void latent_merge(const eagle4_latent_attn_args a, const LatentPlan p) {
  constexpr int LP = RANK / 4, RPB = 256 / LP;
  const uint32_t* const pre = reinterpret_cast<const uint32_t*>(a.workspace + p.pre_off);
  const int at = blockIdx.y, b = p.first + at;
  const uint32_t first = pre[at], total = pre[p.reqs];
  const int rows = static_cast<int>(pre[p.reqs + 1]);  // of a workgroup
  if (pre[at + 1] == first) return;
  const Unit u = unit_of(a, b);
  uint32_t share = (total + p.groups - 1) / p.groups;
  share = share < static_cast<uint32_t>(p.least) ? p.least : share;
  const int rho0 = blockIdx.x * RPB, rg = rho0 / rows;  // rows is a multiple of RPB: one row group
  if (rho0 >= u.width * a.heads) return;
  const uint32_t begin = first + rg * u.tiles, end = begin + u.tiles;
  const int w0 = static_cast<int>(begin / share), w1 = static_cast<int>((end - 1) / share);
  if (w0 == w1) return;
  const int rho = rho0 + threadIdx.x / LP;
  const bool ok = rho < u.width * a.heads;
  f32x4_t sum;
  float wsum;
  merge_partials<RANK, 1>(
      ok ? w1 - w0 + 1 : 0,
      [&](int i) { return (2 * static_cast<int64_t>(w0 + i) + (i == 0 ? 1 : 0)) * rows + (rho - rg * rows); },
      a.workspace + p.part_off, a.workspace + p.lse_off, sum, wsum);
  if (!ok) return;
  const float inv = wsum == 0.f ? 0.f : 1.0f / wsum;
  const int t = rho / a.heads, head = rho % a.heads, d = 4 * (threadIdx.x % LP);
  uint16_t* const o = static_cast<uint16_t*>(a.out) + (u.start + t) * a.stride_ot + head * a.stride_oh + d;
  *reinterpret_cast<u32x2_t*>(o) = u32x2_t{T::pack(sum[0] * inv, sum[1] * inv), T::pack(sum[2] * inv, sum[3] * inv)};
}

constexpr int kGroups = 256;  // one workgroup a CU

bool covered(const eagle4_latent_attn_args& a) {
  const auto tab = [](const eagle4_itab& t) { return t.ptr != nullptr && e4::is_index_dtype(t.dtype); };
  if (a.dtype != EAGLE4_BF16 && a.dtype != EAGLE4_F16) return false;
  if (a.cache_dtype != a.dtype && (a.cache_dtype != EAGLE4_FP8_E4M3 || a.scale_page == nullptr)) return false;
  if ((a.rank != 256 && a.rank != 512) || a.rope != 64) return false;
  if (a.num_reqs < 0 || a.heads < 1 || a.heads > 1024 || a.max_query_len < 1 || a.max_query_len > 64 || a.page < 1 ||
      a.max_blocks < 0 || a.num_blocks < 0)
    return false;
  if (!tab(a.block_table) || a.block_table.dtype != EAGLE4_I32 || a.block_table.s1 != 1 || !tab(a.context_lens) ||
      !tab(a.query_start_loc) || a.masks == nullptr)
    return false;
  // positions are 32-bit, and so are those of the tiles looked up ahead
  if (static_cast<int64_t>(a.max_blocks) * a.page >= (int64_t(1) << 31) - 64 * kKeys) return false;
  for (const int64_t s : {a.stride_qt, a.stride_qh, a.stride_nt, a.stride_cb, a.stride_cs, a.stride_ot, a.stride_oh})
    if (s % 8 != 0) return false;
  if (a.cache_dtype == EAGLE4_FP8_E4M3 && (a.stride_cb % 16 != 0 || a.stride_cs % 16 != 0)) return false;
  for (const void* p : {a.q, a.latent_new, a.cache, static_cast<const void*>(a.out)})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  if (a.tokens > 0 && (a.q == nullptr || a.latent_new == nullptr || a.out == nullptr)) return false;
  if (a.num_blocks > 0 && a.cache == nullptr) return false;
  return true;
}

// Query rows of a workgroup at most: as the widest request's rows fill them.
int rows_of(const eagle4_latent_attn_args& a) {
  const int rows = a.max_query_len * a.heads;
  return rows <= 16 ? 16 : (rows <= 32 ? 32 : 64);
}

// The requests that one launch takes: their tiles (at the most that the tables' sizes allow) are counted in 31 bits.
int reqs_of(const eagle4_latent_attn_args& a, int rows) {
  const int64_t tiles = (static_cast<int64_t>(a.max_blocks) * a.page + kKeys - 1) / kKeys + 2;
  const int64_t most = tiles * e4::ceil_div(static_cast<int64_t>(a.max_query_len) * a.heads, rows);
  const int64_t fit = ((int64_t(1) << 31) - 1 - kGroups * 64) / most;
  return static_cast<int>(fit < 1 ? 0 : (fit < kMaxReqs ? fit : kMaxReqs));
}

LatentPlan plan(const eagle4_latent_attn_args& a) {
  LatentPlan p;
  p.rows = rows_of(a);
  p.groups = kGroups;
  p.least = 2;  // against 4: 16 requests of 4 x 16 rows over 1024 keys 39.4 -> 31.3 us, nothing where runs are longer
  p.first = 0;
  p.page_shift = (a.page & (a.page - 1)) == 0 ? __builtin_ctz(a.page) : -1;
  p.page_inv = a.page > 1 ? static_cast<uint32_t>((uint64_t(1) << 32) / a.page) : 0;
  const int fit = reqs_of(a, p.rows);
  p.reqs = a.num_reqs < fit ? a.num_reqs : fit;
  p.pre_off = 0;
  p.lse_off = (p.reqs + 2 + 3) / 4 * 4;
  p.part_off = p.lse_off + 2 * static_cast<int64_t>(p.groups) * p.rows;
  return p;
}

template <int RANK, typename T, bool FP8>
int launch(const eagle4_latent_attn_args& a, const LatentPlan& p, hipStream_t s) {
  switch (p.rows) {
    case 16: latent_kernel<RANK, 64, T, FP8, 1><<<p.groups, kThreads, 0, s>>>(a, p); break;
    case 32: latent_kernel<RANK, 64, T, FP8, 2><<<p.groups, kThreads, 0, s>>>(a, p); break;
    default: latent_kernel<RANK, 64, T, FP8, 4><<<p.groups, kThreads, 0, s>>>(a, p); break;
  }
  const int status = E4_LAUNCH_STATUS();
  if (status != EAGLE4_OK) return status;
  constexpr int RPB = 1024 / RANK;
  const dim3 grid(e4::ceil_div(int64_t(a.max_query_len) * a.heads, RPB), p.reqs);
  latent_merge<RANK, T><<<grid, 256, 0, s>>>(a, p);
  return E4_LAUNCH_STATUS();
}

template <int RANK>
int launch_rank(const eagle4_latent_attn_args& a, const LatentPlan& p, hipStream_t s) {
  const bool fp8 = a.cache_dtype == EAGLE4_FP8_E4M3;
  if (a.dtype == EAGLE4_BF16) return fp8 ? launch<RANK, e4::Bf16, true>(a, p, s) : launch<RANK, e4::Bf16, false>(a, p, s);
  return fp8 ? launch<RANK, e4::F16, true>(a, p, s) : launch<RANK, e4::F16, false>(a, p, s);
}

}  // namespace

extern "C" int64_t eagle4_latent_attention_workspace(const eagle4_latent_attn_args* a) {
  if (!covered(*a)) return -1;
  if (a->num_reqs == 0) return 0;
  const LatentPlan p = plan(*a);
  if (p.reqs < 1) return -1;
  return (p.part_off + 2 * static_cast<int64_t>(p.groups) * p.rows * a->rank) * static_cast<int64_t>(sizeof(float));
}

extern "C" int eagle4_latent_attention(const eagle4_latent_attn_args* a, void* stream) {
  if (a->num_reqs == 0) return EAGLE4_OK;
  if (!covered(*a) || a->workspace == nullptr || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0 ||
      a->workspace_bytes < eagle4_latent_attention_workspace(a))
    return EAGLE4_NOT_COVERED;
  LatentPlan p = plan(*a);
  if (p.reqs < 1) return EAGLE4_NOT_COVERED;
  const int step = p.reqs;
  for (int first = 0; first < a->num_reqs; first += step) {
    p.first = first;
    p.reqs = a->num_reqs - first < step ? a->num_reqs - first : step;
    const int status = a->rank == 512 ? launch_rank<512>(*a, p, static_cast<hipStream_t>(stream))
                                      : launch_rank<256>(*a, p, static_cast<hipStream_t>(stream));
    if (status != EAGLE4_OK) return status;
  }
  return EAGLE4_OK;
}
