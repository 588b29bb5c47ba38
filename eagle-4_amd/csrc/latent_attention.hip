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
// The launch is one workgroup a CU; each takes an equal run of all (request, row group, tile)s, so requests of any
// lengths fill the chip. A row group cut by a run's end leaves normalised fp32 partials with their log2-sum-exps (at most two
// a workgroup), which a second kernel merges.

#include "attention_tile.h"

namespace {

using namespace e4attn;

constexpr int kKeys = 32;      // keys of a tile
constexpr int kWindow = 256;   // block-table entries held in LDS
constexpr int kMaxReqs = 512; // requests of one launch (their tile counts are kept in LDS)

struct LatentPlan {
  int first, reqs;       // requests of this launch
  int groups;            // workgroups
  int least;             // tiles of a workgroup's run at least
  int rows;              // query rows of a workgroup
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
  int row_groups;
};

E4_DEV Unit unit_of(const eagle4_latent_attn_args& a, int b, int rows) {
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
  u.row_groups = (u.width * a.heads + rows - 1) / rows;
  return u;
}

E4_DEV uint32_t lds_addr(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p));
}
// 64 lanes x 16 bytes from per-lane addresses into LDS [lds, lds + 1024), lane p at lds + 16 p.
E4_DEV void dma16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
template <int N>
E4_DEV void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 8 fp8 codes times a power of two, as 16-bit T (exact but beyond T's range).
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
// as the whole scale would.
E4_DEV void split_scale(float scale, float& pow2, float& rest) {
  const uint32_t e = __float_as_uint(scale) & 0x7f800000u;
  const bool plain = e != 0 && e != 0x7f800000u;
  pow2 = plain ? __uint_as_float(e) : 1.f;
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
// kept in registers over the loop (the 128-row form has none to spare).
E4_DEV int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The bits of lanes 0, 8, .., 56 of a ballot, as a byte; those of lanes 0, 4, .., 60, as 16 bits.
E4_DEV uint8_t every_eighth(uint64_t ballot) {
  return static_cast<uint8_t>(((ballot & 0x0101010101010101ull) * 0x0102040810204080ull) >> 56);
}
E4_DEV uint16_t every_fourth(uint64_t x) {
  x &= 0x1111111111111111ull;
  x = (x | x >> 3) & 0x0303030303030303ull;
  x = (x | x >> 6) & 0x000f000f000f000full;
  x = (x | x >> 12) & 0x000000ff000000ffull;
  return static_cast<uint16_t>(x | x >> 24);
}

// A tile in LDS: CB blocks of 64 columns, each 32 keys x 128 bytes, the eight 16-byte chunks of a key's 128 bytes at
// chunk ^ swz(key). Both operand reads then run at the LDS's full rate (256 bytes a cycle): the scores' (16 keys; the four
// lane groups at chunks 2 g or 2 g + 1) and the transposing one (8 keys at two adjacent chunks). With the lane groups
// at adjacent chunks instead the scores' reads take twice the cycles. An instruction of direct loads fills 8 keys of a block,
// so a lane's address is its key's row plus a constant a block.
E4_DEV int swz(int key) { return 2 * ((key >> 1) & 3) | ((key >> 3) & 1); }

constexpr int kWaves = 8, kThreads = 64 * kWaves;

template <int RANK, int ROPE, typename T_, bool FP8_, int RW_>
struct Shape {
  using T = T_;
  static constexpr bool FP8 = FP8_;
  static constexpr int RW = RW_, DW = kWaves / RW, DT = RANK / 16 / DW;
  static constexpr int DIM = RANK + ROPE, CB = DIM / 64, KC = DIM / 32, ROWS = RW * 16, TILE = CB * 4096;
  // 16-bit pages: a ring of four tiles, two in use and two on their way. fp8 pages: a ring of four tiles of codes, three on
  // their way, and two widened ones.
  static constexpr int NBUF = FP8 ? 2 : 4, RAW = CB * 2048;
  // blocks of 64 columns that waves 0-3 (each 8 keys of a tile) bring in; waves 4-7 bring in the rest
  static constexpr int CB0 = (CB + 1) / 2, CB1 = CB - CB0;
  // LDS operands of the matrix products in registers at a time, the one in use among them. Their loads run that far ahead
  // in this order, product by product: left to itself the compiler waits for each operand right after its load.
  static constexpr int AHEAD = 8;
};

// A wave's share of the weights: P^T of one half tile (16 keys x 16 rows) as written by its lanes, and the rows' maxima.
template <int RW>
struct Weights {
  __attribute__((aligned(16))) u32x2_t p[RW][2][64];
  float m[RW][2][16];
};

// The scores of keys 16 kt .. of a tile, for a wave's 16 rows.
template <typename S>
E4_DEV f32x4_t score_step(const char* tile, const u32x4_t (&q)[S::KC], int kt, int lane) {
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
    __builtin_amdgcn_sched_barrier(0);
  }
  return s[0] + s[1];
}

// The weights of those scores into `to`, relative to the rows' maximum m; l takes their sum. Bit k of bits: key k of the tile
// is visible to the lane's row (`all`: every key to every row).
template <typename S>
E4_DEV void weight_step(f32x4_t s, Weights<S::RW>& to, int row_wave, int kt, bool writes, float& m, float& l,
                        float scale_log2, const float* key_scale, int lane, bool all, uint32_t bits) {
  using T = typename S::T;
  const int g = lane >> 4;
  s *= scale_log2;
  f32x4_t ks = {1.f, 1.f, 1.f, 1.f};
  if constexpr (S::FP8) {
    ks = *reinterpret_cast<const f32x4_t*>(key_scale + 16 * kt + 4 * g);
    s *= ks;
  }
  if (!all) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!((bits >> (16 * kt + 4 * g + i)) & 1)) s[i] = -INFINITY;
  }
  float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
  // The maximum moves only when it grows by more than 2^8 (until then p stays below 2^8, which 16 bits hold as well as
  // values below 1), and to a whole number: what was weighted with the last one is then scaled without rounding.
  if (__any(top > m + 8.f)) {
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float now = fmaxf(m, ceilf(top));
    l *= exp2f(m - now);
    m = now;
  }
  float p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[i] = __builtin_amdgcn_exp2f(s[i] - m);
    l += p[i];
    if constexpr (S::FP8) p[i] *= ks[i];
  }
  if (writes) {
    to.p[row_wave][kt][lane] = u32x2_t{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3])};
    if (g == 0) to.m[row_wave][kt][lane & 15] = m;
  }
}

// Two packed weights times a power of two.
template <typename T>
E4_DEV uint32_t scale2(uint32_t w, float f) {
  return pack2<T>(T::to_f32(static_cast<uint16_t>(w & 0xffffu)) * f, T::to_f32(static_cast<uint16_t>(w >> 16)) * f);
}

// The weights of a tile as the operand of its output. macc is what acc is relative to, m what the wave's own next weights
// are: both move to the largest maximum that the tile's weights bring. (In front of the scores, where no operand of a product
// is in registers: the compiler then keeps one copy of acc over the branch.)
template <typename S>
E4_DEV u32x4_t take_weights(const Weights<S::RW>& from, int row_wave, f32x4_t (&acc)[S::DT], float& macc, float& m, float& l,
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

// O^T += C^T P^T of a tile, for a wave's 16 rows and its columns dbase ...
template <typename S>
E4_DEV void value_step(const char* tile, u32x4_t pb, f32x4_t (&acc)[S::DT], int dbase, int lane) {
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
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int RANK, int ROPE, typename T, bool FP8, int RW>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void latent_kernel(
    const eagle4_latent_attn_args a, const LatentPlan p) {
  using S = Shape<RANK, ROPE, T, FP8, RW>;
  __shared__ __attribute__((aligned(1024))) char smem[S::NBUF][S::TILE];
  __shared__ __attribute__((aligned(1024))) char s_raw[FP8 ? 4 : 1][FP8 ? S::RAW : 16];
  __shared__ Weights<RW> s_w[2];
  __shared__ uint32_t s_pre[kMaxReqs + 1];
  __shared__ int32_t s_win[kWindow];
  __shared__ float s_winscale[FP8 ? kWindow : 1];
  // by tile % 4 (up to three tiles are under way beside the one in use): a bit a key that is there, and its scale's parts
  __shared__ uint32_t s_vis[4];
  __shared__ __attribute__((aligned(16))) float s_rest[4][kKeys], s_pow2[FP8 ? 4 : 1][kKeys];
  __shared__ uint32_t s_bad;           // a bit a new key: it holds a value that is not finite
  __shared__ uint32_t s_tot[kWaves];
  __shared__ float s_sum[RW][2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, l16 = lane & 15;

  // tiles before each request
  uint32_t run = 0;
  for (int b0 = 0; b0 < p.reqs; b0 += kThreads) {
    uint32_t n = 0;
    if (b0 + tid < p.reqs) {
      const Unit u = unit_of(a, p.first + b0 + tid, S::ROWS);
      n = static_cast<uint32_t>(u.tiles) * static_cast<uint32_t>(u.row_groups);
    }
    uint32_t sum = n;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const uint32_t o = __shfl_up(sum, k, 64);
      if (lane >= k) sum += o;
    }
    if (lane == 63) s_tot[wave] = sum;
    __syncthreads();
    uint32_t before = run;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before += s_tot[w];
      run += s_tot[w];
    }
    if (b0 + tid < p.reqs) s_pre[b0 + tid + 1] = before + sum;
    __syncthreads();
  }
  if (tid == 0) s_pre[0] = 0;
  __syncthreads();
  const uint32_t total = uniform(run);
  uint32_t share = (total + p.groups - 1) / p.groups;
  share = share < static_cast<uint32_t>(p.least) ? p.least : share;
  // adjacent runs on one XCD (workgroups go to the eight in turn): row groups of a request share its tiles in the L2
  const int wg = p.groups % 8 == 0 ? (blockIdx.x % 8) * (p.groups / 8) + blockIdx.x / 8 : blockIdx.x;
  if (wg == 0) {  // for the merge
    uint32_t* const pre = reinterpret_cast<uint32_t*>(a.workspace + p.pre_off);
    for (int i = tid; i <= p.reqs; i += kThreads) pre[i] = s_pre[i];
  }
  uint32_t pos = wg * share;
  const uint32_t stop = pos + share < total ? pos + share : total;
  if (pos >= stop) return;
  int at = 0;  // the request of tile `pos`: the last with s_pre <= pos
  for (int step = kMaxReqs / 2; step > 0; step >>= 1)
    if (at + step < p.reqs && uniform(s_pre[at + step]) <= pos) at += step;

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
    while (uniform(s_pre[at + 1]) <= pos) ++at;
    const int b = p.first + at;
    Unit u = unit_of(a, b, S::ROWS);
    u = Unit{uniform(u.start), uniform(u.width), uniform(u.context), uniform(u.ctx_tiles), uniform(u.tiles),
             uniform(u.row_groups)};
    const uint32_t within = pos - uniform(s_pre[at]);
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
    int win0 = 0, win1 = 0;  // the block-table entries in LDS
    const auto window = [&](int tile) {  // makes those of context tile `tile` be there; every thread calls it
      const int lo = uniform(page_of(tile * kKeys));
      const int last = tile * kKeys + kKeys < u.context ? tile * kKeys + kKeys - 1 : u.context - 1;
      if (lo >= win0 && page_of(last) < win1) return;
      __syncthreads();
      win0 = lo;
      win1 = lo + kWindow;
#pragma unroll 1
      for (int i = fresh(tid); i < kWindow; i += kThreads) {
        int32_t blk = -1;
        if (win0 + i < a.max_blocks) blk = table[win0 + i];
        if (blk < 0 || blk >= a.num_blocks) blk = -1;
        s_win[i] = blk;
        if constexpr (FP8) s_winscale[i] = blk >= 0 ? a.scale_page[blk * a.stride_sp] : 0.f;
      }
      __syncthreads();
    };
    // the lane's key row of a tile; null where there is none
    const auto key_row = [&](int tile, int my_key, float& scale) -> const char* {
      scale = 1.f;
      if (tile >= u.ctx_tiles) {
        const int j = (tile - u.ctx_tiles) * kKeys + my_key;
        return j < u.width ? static_cast<const char*>(a.latent_new) + (u.start + j) * a.stride_nt * 2 : nullptr;
      }
      const int k = tile * kKeys + my_key;
      if (k >= u.context) return nullptr;
      const int page = page_of(k);
      const int32_t blk = s_win[page - win0];
      if constexpr (FP8) scale = s_winscale[page - win0];
      return blk >= 0 ? cache + blk * scb + static_cast<int64_t>(k - page * a.page) * scs : nullptr;
    };
    const auto is_ctx = [&](int tile) { return tile < u.ctx_tiles; };
    // a tile of 16-bit rows by direct loads
    const auto issue = [&](int tile) {
      const int ln = fresh(lane), my_key = 8 * octet + ln / 8, my_chunk = (ln % 8) ^ swz(my_key);
      float scale;
      const char* row = key_row(tile, my_key, scale);
      const uint8_t there = every_eighth(__ballot(row != nullptr));
      if (!second_half && ln == 0) reinterpret_cast<uint8_t*>(&s_vis[tile % 4])[octet] = there;
      if (FP8 && !second_half) s_rest[tile % 4][my_key] = 1.f;  // eight lanes, one value
      if (row == nullptr) row = reinterpret_cast<const char*>(zero_row);
      const char* const src = row + 16 * my_chunk + 128 * cb_first;
      const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_addr(smem[tile % S::NBUF]) + 1024 * octet + 4096 * cb_first);
#pragma unroll
      for (int c = 0; c < S::CB1; ++c) dma16(src + 128 * c, dst + 4096 * c);
      if (S::CB0 > S::CB1 && !second_half) dma16(src + 128 * S::CB1, dst + 4096 * S::CB1);
    };
    // a tile of fp8 codes by direct loads: a block of 64 columns is 32 keys x 64 bytes, an instruction 16 keys of it; wave w
    // brings in keys 16 (w % 2) .. of blocks w / 2, w / 2 + kWaves / 2, ..
    const auto issue8 = [&](int tile) {
      const int ln = fresh(lane), my_key = 16 * (wave % 2) + ln / 4;
      float scale, pow2, rest;
      const char* row = key_row(tile, my_key, scale);
      const uint16_t there = every_fourth(__ballot(row != nullptr));
      split_scale(scale, pow2, rest);
      if (wave < 2) {
        if (ln == 0) reinterpret_cast<uint16_t*>(&s_vis[tile % 4])[wave] = there;
        s_pow2[FP8 ? tile % 4 : 0][my_key] = pow2;
        s_rest[tile % 4][my_key] = rest;
      }
      if (row == nullptr) row = reinterpret_cast<const char*>(zero_row);
      const char* const src = row + 16 * (ln % 4);
      const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_addr(s_raw[FP8 ? tile % 4 : 0]) + 1024 * (wave % 2));
#pragma unroll
      for (int c0 = 0; c0 < S::CB; c0 += kWaves / 2)
        if (wave / 2 + c0 < S::CB) dma16(src + 64 * (wave / 2 + c0), dst + 2048 * (wave / 2 + c0));
    };
    const auto widen = [&](int tile) {
      const int ln = fresh(lane), my_key = 8 * octet + ln / 8, my_chunk = (ln % 8) ^ swz(my_key);
      const float pow2 = s_pow2[FP8 ? tile % 4 : 0][my_key];
      const char* const src = s_raw[FP8 ? tile % 4 : 0] + 2048 * cb_first + my_key * 64 + 8 * (ln % 8);
      char* const dst = smem[tile % S::NBUF] + 4096 * cb_first + my_key * 128 + 16 * my_chunk;
      const int blocks = second_half ? S::CB1 : S::CB0;
#pragma unroll
      for (int c = 0; c < S::CB0; ++c)
        if (c < blocks)
          *reinterpret_cast<u32x4_t*>(dst + 4096 * c) = widen8<T>(*reinterpret_cast<const u32x2_t*>(src + 2048 * c), pow2);
    };

    __syncthreads();  // the last piece's tiles have been read
    // the tiles behind the first start after it, so that two (fp8: three) are under way in the loop
    const auto start = [&](int tile) {
      if (tile >= t1 || (FP8 && !is_ctx(tile))) return;
      if constexpr (FP8) issue8(tile); else issue(tile);
    };
#pragma unroll 1
    for (int i = 0; i < (FP8 ? 3 : 2); ++i) {
      if (t0 + i < t1 && is_ctx(t0 + i)) window(t0 + i);
      start(t0 + i);
    }
    // Waits until a tile (fp8: its codes) is there for every wave, the last tile's weights too; the buffer of the tile before
    // that is free.
    const auto arrive = [&](int tile) {
      if constexpr (FP8) {
        // instructions a tile of waves below 2 (CB % 4); the others one less
        constexpr int kMost = (S::CB + 3) / 4;
        const bool less = S::CB % 4 != 0 && wave >= 2 * (S::CB % 4);
        if (tile + 2 < t1 && is_ctx(tile + 2)) {
          if (less) wait_vm<2 * (kMost - 1)>(); else wait_vm<2 * kMost>();
        } else if (tile + 1 < t1 && is_ctx(tile + 1)) {
          if (less) wait_vm<kMost - 1>(); else wait_vm<kMost>();
        } else {
          wait_vm<0>();
        }
      } else {
        if (tile + 1 < t1) {
          if (second_half) wait_vm<S::CB1>(); else wait_vm<S::CB0>();
        } else {
          wait_vm<0>();
        }
      }
      __syncthreads();
    };
    // The round's rows. One that is not finite must not reach the rows that do not see it through 0 x NaN: it is cleared, and
    // the rows that see it become NaN. Gives a bit a row that was cleared; every wave calls it.
    const auto clean = [&](int tile) {
      if (tid == 0) s_bad = 0;
      __syncthreads();
      const int ln = fresh(lane), my_key = 8 * octet + ln / 8;
      char* const mine = smem[tile % S::NBUF] + 4096 * cb_first + my_key * 128 + 16 * (ln % 8);
      bool bad = false;
#pragma unroll 1
      for (int c = 0; c < (second_half ? S::CB1 : S::CB0); ++c) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(mine + 4096 * c);
        constexpr uint32_t kExp = T::code == EAGLE4_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= (w[i] & kExp) == kExp || ((w[i] >> 16) & kExp) == kExp;
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
    // The first iteration's output: no weights over a tile of zeros.
    for (int i = tid; i < S::TILE / 16; i += kThreads)
      *reinterpret_cast<u32x4_t*>(smem[(t0 + S::NBUF - 1) % S::NBUF] + 16 * i) = u32x4_t{0u, 0u, 0u, 0u};
    if (tid < RW * 64) {
      s_w[(t0 + 1) % 2].p[tid / 64][0][lane] = s_w[(t0 + 1) % 2].p[tid / 64][1][lane] = u32x2_t{0u, 0u};
      if (lane < 32) s_w[(t0 + 1) % 2].m[tid / 64][lane / 16][l16] = kNone;
    }
    // What every wave does in iteration `tile`, before its products and after: the tile's arrival, the loads of a later one.
    const auto begin = [&](int tile) {
      arrive(tile);
      const int ahead = tile + (FP8 ? 3 : 2);
      if (ahead < t1 && is_ctx(ahead)) window(ahead);
      // 16-bit pages: waves 0-3 start the tile two ahead before their products, waves 4-7 after, so that of the two waves
      // of a SIMD one has the matrix cores while the other is at its loads.
      if (FP8 || !second_half) start(ahead);
      if (FP8 && tile < t1) {
        if (is_ctx(tile)) widen(tile);
        else issue(tile);  // the round's rows are 16-bit: brought in here, there are few of them
      }
    };
    const auto widened = [&](int tile) {
      if (!is_ctx(tile)) wait_vm<0>();
      __syncthreads();
    };
    if (!computes) {  // no rows of this row group: a share of the loads alone
      for (int tile = t0; tile <= t1; ++tile) {
        begin(tile);
        if (FP8 && tile < t1) widened(tile);
        if (tile < t1 && !is_ctx(tile)) clean(tile);
        if (!FP8 && second_half) start(tile + 2);
      }
      __syncthreads();
      pos += t1 - t0;
      continue;
    }
    u32x4_t q[S::KC];
    f32x4_t acc[S::DT];
    float m = kNone, macc = kNone, l = 0.f;
#pragma unroll
    for (int dt = 0; dt < S::DT; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    {
      int rho, t, head;
      const bool ok = my_row(rho, t, head);
      const uint16_t* const qrow = static_cast<const uint16_t*>(a.q) + (u.start + t) * a.stride_qt + head * a.stride_qh;
#pragma unroll
      for (int c = 0; c < S::KC; ++c)  // the columns of the lane's chunk of the scores' operand
        q[c] = ok ? *reinterpret_cast<const u32x4_t*>(qrow + 64 * (c / 2) + 8 * (2 * g + (c & 1))) : u32x4_t{0u, 0u, 0u, 0u};
      // Settled here, once: a wait for them inside the loop would wait for the tiles on their way too.
#pragma unroll
      for (int c = 0; c < S::KC; ++c) asm volatile("" : "+v"(q[c]));
    }
    // Iteration `tile`: its scores and weights, and the output of the tile before it.
    for (int tile = t0; tile <= t1; ++tile) {
      begin(tile);
      uint32_t bits = 0xffffffffu;
      bool all = true;
      f32x4_t s = {0.f, 0.f, 0.f, 0.f};
      const auto score = [&] {
        const uint32_t vis = __builtin_amdgcn_readfirstlane(s_vis[tile % 4]);
        bits = vis;
        all = is_ctx(tile) && vis == 0xffffffffu;
        if (!is_ctx(tile)) {
          const uint32_t poison = clean(tile);
          int rho, t, head;
          const uint64_t mask = my_row(rho, t, head) ? static_cast<uint64_t>(a.masks[b * a.stride_mask + t]) : 0;
          bits = static_cast<uint32_t>(mask >> ((tile - u.ctx_tiles) * kKeys)) & vis;
          if (bits & poison) l = __builtin_nanf("");
        }
        s = score_step<S>(smem[tile % S::NBUF], q, kt, fresh(lane));
      };
      const u32x4_t pb = take_weights<S>(s_w[(tile + 1) % 2], row_wave, acc, macc, m, l, fresh(lane));
      if (!FP8 && tile < t1) score();
      value_step<S>(smem[(tile + S::NBUF - 1) % S::NBUF], pb, acc, dbase, fresh(lane));
      if (FP8 && tile < t1) {
        widened(tile);
        score();
      }
      if (tile < t1)
        weight_step<S>(s, s_w[tile % 2], row_wave, kt, column_wave < 2, m, l, scale_log2, s_rest[tile % 4], fresh(lane), all,
                       bits);
      if (!FP8 && second_half) start(tile + 2);
    }
    // the sum over both halves of the keys: each wave's own is relative to the last maximum by now
    float sum = l + __shfl_xor(l, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (column_wave < 2 && g == 0) s_sum[row_wave][kt][l16] = sum;
    __syncthreads();
    sum = s_sum[row_wave][0][l16] + s_sum[row_wave][1][l16];

    const bool whole = t0 == 0 && t1 == u.tiles;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // nothing seen: zeros
    int rho, t, head;
    const bool ok = my_row(rho, t, head);
    if (ok && whole) {
      uint16_t* const o = static_cast<uint16_t*>(a.out) + (u.start + t) * a.stride_ot + head * a.stride_oh + dbase;
#pragma unroll
      for (int dt = 0; dt < S::DT; ++dt)
        *reinterpret_cast<u32x2_t*>(o + 16 * dt + 4 * g) =
            u32x2_t{pack2<T>(acc[dt][0] * inv, acc[dt][1] * inv), pack2<T>(acc[dt][2] * inv, acc[dt][3] * inv)};
    } else if (ok) {
      const int64_t part = (2 * static_cast<int64_t>(wg) + (t0 == 0 ? 1 : 0)) * S::ROWS + rho - rg * S::ROWS;
      float* const o = a.workspace + p.part_off + part * RANK + dbase;
#pragma unroll
      for (int dt = 0; dt < S::DT; ++dt) *reinterpret_cast<f32x4_t*>(o + 16 * dt + 4 * g) = acc[dt] * inv;
      if (g == 0 && dbase == 0) a.workspace[p.lse_off + part] = sum == 0.f ? -INFINITY : macc + log2f(sum);
    }
    pos += t1 - t0;
  }
}

// Rows of row groups that were cut: their partials by log2-sum-exp. One workgroup per 2 / SG rows.
template <int RANK, int SG, typename T>
__global__ __launch_bounds__(256) void latent_merge(const eagle4_latent_attn_args a, const LatentPlan p) {
  constexpr int LP = RANK / 4, RPB = 256 / LP / SG;
  const uint32_t* const pre = reinterpret_cast<const uint32_t*>(a.workspace + p.pre_off);
  const int at = blockIdx.y, b = p.first + at;
  const uint32_t first = pre[at], total = pre[p.reqs];
  if (pre[at + 1] == first) return;
  const Unit u = unit_of(a, b, p.rows);
  uint32_t share = (total + p.groups - 1) / p.groups;
  share = share < static_cast<uint32_t>(p.least) ? p.least : share;
  const int rho0 = blockIdx.x * RPB, rg = rho0 / p.rows;  // p.rows is a multiple of RPB: one row group
  if (rho0 >= u.width * a.heads) return;
  const uint32_t begin = first + rg * u.tiles, end = begin + u.tiles;
  const int w0 = static_cast<int>(begin / share), w1 = static_cast<int>((end - 1) / share);
  if (w0 == w1) return;
  const int rho = rho0 + threadIdx.x / (LP * SG);
  const bool ok = rho < u.width * a.heads;
  f32x4_t sum;
  float wsum;
  const bool mine = merge_partials<RANK, SG>(
      ok ? w1 - w0 + 1 : 0,
      [&](int i) { return (2 * static_cast<int64_t>(w0 + i) + (i == 0 ? 1 : 0)) * p.rows + (rho - rg * p.rows); },
      a.workspace + p.part_off, a.workspace + p.lse_off, sum, wsum);
  if (!mine || !ok) return;
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
  if (static_cast<int64_t>(a.max_blocks) * a.page >= (int64_t(1) << 31) - kKeys) return false;  // 32-bit positions
  for (const int64_t s : {a.stride_qt, a.stride_qh, a.stride_nt, a.stride_cb, a.stride_cs, a.stride_ot, a.stride_oh})
    if (s % 8 != 0) return false;
  if (a.cache_dtype == EAGLE4_FP8_E4M3 && (a.stride_cb % 16 != 0 || a.stride_cs % 16 != 0)) return false;
  for (const void* p : {a.q, a.latent_new, a.cache, static_cast<const void*>(a.out)})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  return true;
}

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
  p.least = 4;
  p.first = 0;
  p.page_shift = (a.page & (a.page - 1)) == 0 ? __builtin_ctz(a.page) : -1;
  p.page_inv = a.page > 1 ? static_cast<uint32_t>((uint64_t(1) << 32) / a.page) : 0;
  const int fit = reqs_of(a, p.rows);
  p.reqs = a.num_reqs < fit ? a.num_reqs : fit;
  p.pre_off = 0;
  p.lse_off = (p.reqs + 1 + 3) / 4 * 4;
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
  latent_merge<RANK, 1, T><<<grid, 256, 0, s>>>(a, p);
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
