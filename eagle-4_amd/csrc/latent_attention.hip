// Tree-verify attention over latent rows on gfx950: every head's key is a token's cached row c of RANK + ROPE values, its
// value the row's first RANK.
//
// Mathematics. For a query row (draft token, head): o = sum_k softmax_k(scale q . c_k) c_k[0..RANK), keys the request's
// context and the round's rows in the draft token's ancestor mask. One pass with a running maximum and sum (log2 domain).
//
// What bounds it. A request's width x heads query rows share every key: 2 (2 RANK + ROPE) operations a row and key against
// 2 (RANK + ROPE) bytes a key (16-bit pages). From about 128 rows on that is the matrix cores' work, below it HBM's.
//
// Split. A workgroup takes ROWS query rows (16 to 128) and a run of 32-key tiles, which all four waves read from LDS:
//   - RW row waves of NR 16-row tiles each; the 4 / RW waves of the same rows share out the output's columns (and
//     compute the scores each for itself: with few rows the matrix cores have time for it);
//   - S^T = C Q^T on v_mfma_f32_16x16x32, so that a lane holds scores of one query row, P^T is the B operand of
//     O^T = C^T P^T straight from registers, and C^T is read by transposing LDS loads of the same tile: a row of the
//     cache is brought in once for both products;
//   - the output (RANK columns of fp32 a row) stays in registers: 128 rows take 256 registers a lane, so one wave a SIMD.
// The launch is one workgroup a CU; each takes an equal run of all (request, row group, tile)s, so requests of any
// lengths fill the chip. A row group cut by a run's end leaves normalised fp32 partials with their log2-sum-exps (at most two
// a workgroup), which a second kernel merges.

#include "attention_tile.h"

namespace {

using namespace e4attn;

constexpr int kKeys = 32;      // keys of a tile
constexpr int kWindow = 1024;  // block-table entries held in LDS
constexpr int kMaxReqs = 2048; // requests of one launch (their tile counts are kept in LDS)

struct LatentPlan {
  int first, reqs;       // requests of this launch
  int groups;            // workgroups
  int least;             // tiles of a workgroup's run at least
  int rows;              // query rows of a workgroup
  int64_t pre_off, lse_off, part_off;  // float offsets into the workspace
};

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

// The bits of lanes 0, 8, .., 56 of a ballot, as a byte.
E4_DEV uint8_t every_eighth(uint64_t ballot) {
  return static_cast<uint8_t>(((ballot & 0x0101010101010101ull) * 0x0102040810204080ull) >> 56);
}

// A tile in LDS: CB blocks of 64 columns, each 32 keys x 128 bytes, the eight 16-byte chunks of a key's 128 bytes at
// chunk ^ swz(key). 16 keys at one chunk (the scores' operand) and 8 keys at two adjacent chunks (the transposing
// reads) then fall on distinct banks; an instruction of direct loads fills 8 keys of a block, so a lane's address is
// its key's row plus a constant a block.
E4_DEV int swz(int key) { return 2 * ((key >> 1) & 3) | ((key >> 3) & 1); }

template <int RANK, int ROPE, typename T, bool FP8, int RW, int NR>
struct Shape {
  static constexpr int DIM = RANK + ROPE, CB = DIM / 64, KC = DIM / 32, DW = 4 / RW, DT = RANK / 16 / DW;
  static constexpr int ROWS = RW * NR * 16, TILE = CB * 4096;
  static constexpr int NBUF = FP8 ? 2 : 4;
};

// One tile for a wave's NR x 16 rows; bit k of bits[r]: key k is visible to the lane's row r (`all`: every key to all).
template <typename S, int NR, typename T, bool FP8>
E4_DEV void tile_step(const char* tile, const u32x4_t (&q)[NR][S::KC], f32x4_t (&acc)[NR][S::DT], float (&m)[NR],
                      float (&l)[NR], float scale_log2, const float* key_scale, int dbase, int g, int l16, bool all,
                      const uint32_t (&bits)[NR]) {
  f32x4_t s[NR][2];
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) s[r][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int x = swz(l16);
  const char* const k0 = tile + l16 * 128 + 16 * (g ^ x);
  const char* const k1 = tile + l16 * 128 + 16 * ((4 + g) ^ x);
#pragma unroll
  for (int c = 0; c < S::KC; ++c) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const u32x4_t ka = *reinterpret_cast<const u32x4_t*>((c & 1 ? k1 : k0) + (c / 2) * 4096 + kt * 2048);
#pragma unroll
      for (int r = 0; r < NR; ++r) s[r][kt] = mfma16<T>(ka, q[r][c], s[r][kt]);
    }
    if (c % 3 == 2) __builtin_amdgcn_sched_barrier(0);
  }
  float ks[2][4];
  if constexpr (FP8) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(key_scale + 16 * kt + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) ks[kt][i] = v[i];
    }
  }
  u32x4_t pb[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = s[r][kt][i] * scale_log2;
        if constexpr (FP8) v *= ks[kt][i];
        if (!all) v = (bits[r] >> (16 * kt + 4 * g + i)) & 1 ? v : -INFINITY;
        s[r][kt][i] = v;
        top = fmaxf(top, v);
      }
    }
    // The maximum moves only when it grows by more than 2^8: until then p stays below 2^8, which 16 bits hold as well
    // as values below 1, and the output (up to 256 registers) is not rescaled.
    if (__any(top > m[r] + 8.f)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float now = fmaxf(m[r], top);
      const float keep = exp2f(m[r] - now);
      m[r] = now;
      l[r] *= keep;
#pragma unroll
      for (int dt = 0; dt < S::DT; ++dt) acc[r][dt] *= keep;
    }
    uint32_t w[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {  // element i of P^T's operand is key 16 (i / 4) + 4 g + i % 4
      float p0 = __builtin_amdgcn_exp2f(s[r][p >> 1][2 * (p & 1)] - m[r]);
      float p1 = __builtin_amdgcn_exp2f(s[r][p >> 1][2 * (p & 1) + 1] - m[r]);
      l[r] += p0 + p1;
      if constexpr (FP8) {
        p0 *= ks[p >> 1][2 * (p & 1)];
        p1 *= ks[p >> 1][2 * (p & 1) + 1];
      }
      w[p] = pack2<T>(p0, p1);
    }
    pb[r] = u32x4_t{w[0], w[1], w[2], w[3]};
  }
  const int j = l16 >> 2, s4 = l16 & 3, kv = 4 * g + j, xv = swz(kv);
  const char* const vrow = tile + kv * 128 + 8 * (s4 & 1);
#pragma unroll
  for (int dt = 0; dt < S::DT; ++dt) {
    // columns dbase + 16 dt ..: block (dbase / 64) + dt / 4, chunks 2 (dt % 4) and the next (dbase is a multiple of 64)
    const char* const at = vrow + (dbase / 64 + dt / 4) * 4096 + 16 * ((2 * (dt & 3) + (s4 >> 1)) ^ xv);
    const v4i16 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(at));
    const v4i16 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(at + 2048));
    const u32x2_t lo = __builtin_bit_cast(u32x2_t, lo4), hi = __builtin_bit_cast(u32x2_t, hi4);
    const u32x4_t va = u32x4_t{lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
    for (int r = 0; r < NR; ++r) acc[r][dt] = mfma16<T>(va, pb[r], acc[r][dt]);
    if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
  }
}

template <int RANK, int ROPE, typename T, bool FP8, int RW, int NR>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void latent_kernel(
    const eagle4_latent_attn_args a, const LatentPlan p) {
  using S = Shape<RANK, ROPE, T, FP8, RW, NR>;
  __shared__ __attribute__((aligned(1024))) char smem[S::NBUF][S::TILE];
  __shared__ uint32_t s_pre[kMaxReqs + 1];
  __shared__ int32_t s_win[kWindow];
  __shared__ float s_winscale[FP8 ? kWindow : 1];
  __shared__ __attribute__((aligned(16))) float s_ks[S::NBUF][kKeys];
  __shared__ uint32_t s_vis[S::NBUF];  // a bit a key: it is there
  __shared__ uint32_t s_bad;           // a bit a new key: it holds a value that is not finite
  __shared__ uint32_t s_tot[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, l16 = lane & 15;

  // tiles before each request
  uint32_t run = 0;
  for (int b0 = 0; b0 < p.reqs; b0 += 256) {
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
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += s_tot[w];
      run += s_tot[w];
    }
    if (b0 + tid < p.reqs) s_pre[b0 + tid + 1] = before + sum;
    __syncthreads();
  }
  if (tid == 0) s_pre[0] = 0;
  __syncthreads();
  const uint32_t total = run;
  uint32_t share = (total + p.groups - 1) / p.groups;
  share = share < static_cast<uint32_t>(p.least) ? p.least : share;
  // adjacent runs on one XCD (workgroups go to the eight in turn): row groups of a request share its tiles in the L2
  const int wg = p.groups % 8 == 0 ? (blockIdx.x % 8) * (p.groups / 8) + blockIdx.x / 8 : blockIdx.x;
  if (wg == 0) {  // for the merge
    uint32_t* const pre = reinterpret_cast<uint32_t*>(a.workspace + p.pre_off);
    for (int i = tid; i <= p.reqs; i += 256) pre[i] = s_pre[i];
  }
  uint32_t pos = wg * share;
  const uint32_t stop = pos + share < total ? pos + share : total;
  if (pos >= stop) return;
  int at = 0;  // the request of tile `pos`: the last with s_pre <= pos
  for (int step = 1 << 11; step > 0; step >>= 1)
    if (at + step < p.reqs && s_pre[at + step] <= pos) at += step;

  const int row_wave = wave / S::DW, dbase = (wave % S::DW) * S::DT * 16;
  const float scale_log2 = a.scale * 1.4426950408889634f;
  constexpr int EB = FP8 ? 1 : 2;
  const char* const cache = static_cast<const char*>(a.cache);
  const int64_t scb = a.stride_cb * EB, scs = a.stride_cs * EB;
  const int page_shift = (a.page & (a.page - 1)) == 0 ? __builtin_ctz(a.page) : -1;
  const auto page_of = [&](int pos) {
    return page_shift >= 0 ? pos >> page_shift
                           : static_cast<int>(static_cast<uint32_t>(pos) / static_cast<uint32_t>(a.page));
  };
  // this lane's key of a tile and where its chunks go: a wave brings in 8 keys, 8 lanes a key
  const int my_key = 8 * wave + lane / 8;
  const int my_chunk = (lane % 8) ^ swz(my_key);

  while (pos < stop) {
    while (s_pre[at + 1] <= pos) ++at;
    const int b = p.first + at;
    const Unit u = unit_of(a, b, S::ROWS);
    const uint32_t within = pos - s_pre[at];
    const int rg = static_cast<int>(within / u.tiles), t0 = static_cast<int>(within % u.tiles);
    const int t1 = static_cast<int>(static_cast<uint32_t>(u.tiles - t0) < stop - pos ? u.tiles : t0 + (stop - pos));
    const int32_t* const table = static_cast<const int32_t*>(a.block_table.ptr) + b * a.block_table.s0;

    u32x4_t q[NR][S::KC];
    f32x4_t acc[NR][S::DT];
    float m[NR], l[NR];
    uint64_t mask[NR];
    int rho[NR];
    bool ok[NR], computes = false;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      rho[r] = rg * S::ROWS + (row_wave * NR + r) * 16 + l16;
      ok[r] = rho[r] < u.width * a.heads;
      computes |= rg * S::ROWS + (row_wave * NR + r) * 16 < u.width * a.heads;
      const int t = ok[r] ? rho[r] / a.heads : 0, head = ok[r] ? rho[r] % a.heads : 0;
      const uint16_t* const qrow = static_cast<const uint16_t*>(a.q) + (u.start + t) * a.stride_qt + head * a.stride_qh;
#pragma unroll
      for (int c = 0; c < S::KC; ++c)
        q[r][c] = ok[r] ? *reinterpret_cast<const u32x4_t*>(qrow + 32 * c + 8 * g) : u32x4_t{0u, 0u, 0u, 0u};
      mask[r] = ok[r] ? static_cast<uint64_t>(a.masks[b * a.stride_mask + t]) : 0;
      m[r] = -3.0e38f;
      l[r] = 0.f;
#pragma unroll
      for (int dt = 0; dt < S::DT; ++dt) acc[r][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    int win0 = 0, win1 = 0;  // the block-table entries in LDS
    const auto window = [&](int tile) {  // makes those of context tile `tile` be there; every thread calls it
      const int lo = page_of(tile * kKeys);
      const int last = tile * kKeys + kKeys < u.context ? tile * kKeys + kKeys - 1 : u.context - 1;
      if (lo >= win0 && page_of(last) < win1) return;
      __syncthreads();
      win0 = lo;
      win1 = lo + kWindow;
      for (int i = tid; i < kWindow; i += 256) {
        int32_t blk = -1;
        if (win0 + i < a.max_blocks) blk = table[win0 + i];
        if (blk < 0 || blk >= a.num_blocks) blk = -1;
        s_win[i] = blk;
        if constexpr (FP8) s_winscale[i] = blk >= 0 ? a.scale_page[blk * a.stride_sp] : 0.f;
      }
      __syncthreads();
    };
    // the lane's key row of a tile; null where there is none
    const auto key_row = [&](int tile, float& scale) -> const char* {
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
    const auto mark = [&](int buf, bool there, float scale) {
      const uint8_t byte = every_eighth(__ballot(there));
      if (lane == 0) reinterpret_cast<uint8_t*>(&s_vis[buf])[wave] = byte;
      if (FP8 && lane % 8 == 0) s_ks[buf][my_key] = scale;
    };
    // a tile of 16-bit rows by direct loads
    const auto issue = [&](int tile, int buf) {
      float scale;
      const char* row = key_row(tile, scale);
      mark(buf, row != nullptr, 1.f);
      if (row == nullptr) row = reinterpret_cast<const char*>(zero_row);
      const char* const src = row + 16 * my_chunk;
      const uint32_t dst = lds_addr(smem[buf]) + 1024 * wave;
#pragma unroll
      for (int c = 0; c < S::CB; ++c) dma16(src + 128 * c, dst + 4096 * c);
    };
    // a tile of fp8 rows through registers: raw codes now, widened into LDS a tile later
    u32x2_t raw[FP8 ? S::CB : 1];
    float raw_scale = 1.f;
    bool raw_there = false;
    const auto load8 = [&](int tile) {
      const char* const row = key_row(tile, raw_scale);
      raw_there = row != nullptr;
#pragma unroll
      for (int c = 0; c < S::CB; ++c)
        raw[FP8 ? c : 0] = raw_there ? *reinterpret_cast<const u32x2_t*>(row + 64 * c + 8 * (lane % 8)) : u32x2_t{0u, 0u};
    };
    const auto store8 = [&](int buf) {
      float pow2, rest;
      split_scale(raw_scale, pow2, rest);
      mark(buf, raw_there, rest);
#pragma unroll
      for (int c = 0; c < S::CB; ++c)
        *reinterpret_cast<u32x4_t*>(smem[buf] + 4096 * c + my_key * 128 + 16 * my_chunk) =
            widen8<T>(raw[FP8 ? c : 0], pow2);
    };
    const auto is_ctx = [&](int tile) { return tile < u.ctx_tiles; };

    __syncthreads();  // the last piece's tiles have been read
    if constexpr (FP8) {
      if (is_ctx(t0)) {
        window(t0);
        load8(t0);
        store8(t0 & 1);
      } else {
        issue(t0, t0 & 1);
      }
      if (t0 + 1 < t1 && is_ctx(t0 + 1)) {
        window(t0 + 1);
        load8(t0 + 1);
      }
    } else {
      for (int i = 0; i < S::NBUF - 1 && t0 + i < t1; ++i) {
        if (is_ctx(t0 + i)) window(t0 + i);
        issue(t0 + i, (t0 + i) % S::NBUF);
      }
    }
    for (int tile = t0; tile < t1; ++tile) {
      const int buf = tile % S::NBUF;
      if constexpr (FP8) {
        wait_vm<0>();
      } else {
        if (tile + 2 < t1)
          wait_vm<2 * S::CB>();
        else if (tile + 1 < t1)
          wait_vm<S::CB>();
        else
          wait_vm<0>();
      }
      __syncthreads();  // the tile is there for every wave, and the buffer of the last one is free
      if constexpr (FP8) {
        if (tile + 1 < t1) {
          if (is_ctx(tile + 1))
            store8((tile + 1) & 1);
          else
            issue(tile + 1, (tile + 1) & 1);
        }
        if (tile + 2 < t1 && is_ctx(tile + 2)) {
          window(tile + 2);
          load8(tile + 2);
        }
      } else {
        const int ahead = tile + S::NBUF - 1;
        if (ahead < t1) {
          if (is_ctx(ahead)) window(ahead);
          issue(ahead, ahead % S::NBUF);
        }
      }
      const char* const data = smem[buf];
      const uint32_t vis = __builtin_amdgcn_readfirstlane(s_vis[buf]);
      uint32_t bits[NR];
      if (is_ctx(tile)) {
#pragma unroll
        for (int r = 0; r < NR; ++r) bits[r] = vis;
      } else {
        // The round's rows. One that is not finite must not reach the rows that do not see it through 0 x NaN: it is
        // cleared, and the rows that see it become NaN.
        bool bad = false;
        char* const mine = smem[buf] + my_key * 128 + 16 * (lane % 8);
#pragma unroll 1
        for (int c = 0; c < S::CB; ++c) {
          const u32x4_t w = *reinterpret_cast<const u32x4_t*>(mine + 4096 * c);
          constexpr uint32_t kExp = T::code == EAGLE4_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
          for (int i = 0; i < 4; ++i) bad |= (w[i] & kExp) == kExp || ((w[i] >> 16) & kExp) == kExp;
        }
        uint64_t any = __ballot(bad);
        any |= any >> 4;
        any |= any >> 2;
        any |= any >> 1;
        const uint8_t byte = every_eighth(any);
        if (lane == 0) reinterpret_cast<uint8_t*>(&s_bad)[wave] = byte;
        if ((byte >> (lane / 8)) & 1) {
#pragma unroll 1
          for (int c = 0; c < S::CB; ++c) *reinterpret_cast<u32x4_t*>(mine + 4096 * c) = u32x4_t{0u, 0u, 0u, 0u};
        }
        __syncthreads();
        const uint32_t poison = __builtin_amdgcn_readfirstlane(s_bad);
        const int first_new = (tile - u.ctx_tiles) * kKeys;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          bits[r] = static_cast<uint32_t>(mask[r] >> first_new) & vis;
          if (bits[r] & poison) l[r] = __builtin_nanf("");
        }
      }
      if (computes)
        tile_step<S, NR, T, FP8>(data, q, acc, m, l, scale_log2, s_ks[buf], dbase, g, l16,
                                 is_ctx(tile) && vis == 0xffffffffu, bits);
    }

    const bool whole = t0 == 0 && t1 == u.tiles;
    const int64_t slot = 2 * static_cast<int64_t>(wg) + (t0 == 0 ? 1 : 0);
    if (computes) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float sum = l[r] + __shfl_xor(l[r], 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // nothing seen: zeros
        if (!ok[r]) continue;
        if (whole) {
          const int t = rho[r] / a.heads, head = rho[r] % a.heads;
          uint16_t* const o = static_cast<uint16_t*>(a.out) + (u.start + t) * a.stride_ot + head * a.stride_oh + dbase;
#pragma unroll
          for (int dt = 0; dt < S::DT; ++dt)
            *reinterpret_cast<u32x2_t*>(o + 16 * dt + 4 * g) =
                u32x2_t{pack2<T>(acc[r][dt][0] * inv, acc[r][dt][1] * inv), pack2<T>(acc[r][dt][2] * inv, acc[r][dt][3] * inv)};
        } else {
          const int64_t part = slot * S::ROWS + rho[r] - rg * S::ROWS;
          float* const o = a.workspace + p.part_off + part * RANK + dbase;
#pragma unroll
          for (int dt = 0; dt < S::DT; ++dt) *reinterpret_cast<f32x4_t*>(o + 16 * dt + 4 * g) = acc[r][dt] * inv;
          if (g == 0 && dbase == 0) a.workspace[p.lse_off + part] = sum == 0.f ? -INFINITY : m[r] + log2f(sum);
        }
      }
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
    case 16: latent_kernel<RANK, 64, T, FP8, 1, 1><<<p.groups, 256, 0, s>>>(a, p); break;
    case 32: latent_kernel<RANK, 64, T, FP8, 1, 2><<<p.groups, 256, 0, s>>>(a, p); break;
    default: latent_kernel<RANK, 64, T, FP8, 2, 2><<<p.groups, 256, 0, s>>>(a, p); break;
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
