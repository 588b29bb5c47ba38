// Block tables that follow the requests' lengths, and the cache slots of a batch's rows, on gfx950: whole numbers only, so
// that neither a host's allocator nor its tables are on a round's path.
//
// eagle4_resize_tables: one workgroup. The stack of free pages is one sequence, so which entries a request gives or takes follows
// from running sums over the batch; a chunk of 1024 requests has its sums in LDS, and the threads take the pages that move, finding
// the request of a page by its place in the sums. What bounds a round is latency: loads that depend on each other (slots and
// lengths, page counts, then the pages of both directions). 64 requests by a few pages, up and back with both maps of their
// rows, take 15.3 us in a graph. Where many pages move it is this one workgroup's searches, in proportion to the pages (65 thousand of them
// 103 us, below): there a launch for the sums and one of many workgroups for the moves would be faster. It is not built.
//
// eagle4_slot_maps: some workgroups a request, each with its share of the request's rows and table entries; no row is searched for.

#include "common.h"

namespace {

constexpr int NT = 1024;

struct Chunk {
  int32_t slot[NT], from[NT];  // a request's state slot; its first page that moves
  uint32_t ends[NT];           // running sums of the pages that move
  uint32_t part[NT / 64];
};

// Inclusive running sum over the workgroup.
E4_DEV uint32_t block_scan(uint32_t x, uint32_t* part, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(x, d, 64);
    if (lane >= d) x += o;
  }
  __syncthreads();
  if (lane == 63) part[wave] = x;
  __syncthreads();
  for (int i = 0; i < wave; ++i) x += part[i];
  return x;
}

struct Request {
  int64_t slot;  // negative: none
  int have, need;
};

E4_DEV Request request_of(const eagle4_resize_tables_args& a, int r) {
  Request q{-1, 0, 0};
  if (r >= a.num_reqs) return q;
  const int64_t slot = e4::ld(a.idx_mapping, r), len = e4::ld(a.lens, r);
  if (slot < 0 || slot >= a.slots) return q;
  const int held = a.num_pages[slot];
  q.slot = slot;
  q.have = held < 0 ? 0 : held < a.max_pages ? held : a.max_pages;
  const int64_t need = len > 0 ? (len - 1) / a.page + 1 : 0;
  q.need = need <= a.max_pages ? static_cast<int>(need) : q.have;
  return q;
}

// Moves this thread's pages of the chunk's `all`: load and store get a page's number in the chunk, its request, and its number among
// the request's that move. The search's LDS reads are most of it where many move: 512 prompts' 65 thousand pages, up, mapped and
// back, take 103 us, and 122 with a loop that ends when the request is found.
static_assert(NT == 1 << 10, "ten steps of the search");
template <typename Load, typename Store>
E4_DEV void move_pages(const Chunk& c, uint32_t all, int tid, Load&& load, Store&& store) {
  for (uint32_t f = tid; f < all; f += NT) {
    int lo = 0, hi = NT - 1;  // the first request whose running sum passes f: ten steps, and once found it stays
#pragma unroll
    for (int step = 0; step < 10; ++step) {
      const int mid = (lo + hi) >> 1;
      const bool past = c.ends[mid] > f;
      hi = past ? mid : hi;
      lo = past ? lo : mid + 1;
    }
    const int i = static_cast<int>(f - (lo > 0 ? c.ends[lo - 1] : 0));
    store(f, lo, i, load(f, lo, i));
  }
}

__global__ __launch_bounds__(NT) void resize_tables_kernel(const eagle4_resize_tables_args a) {
  __shared__ Chunk c;
  __shared__ int64_t s_total;
  __shared__ uint32_t s_served;
  const int tid = threadIdx.x;
  const int chunks = (a.num_reqs + NT - 1) / NT;
  const int64_t before = *a.num_free;
  // what comes back in all (the requests of a batch of one chunk are looked up once)
  const Request first = request_of(a, tid);
  int64_t back = 0;
  for (int i = 0; i < chunks; ++i) {
    const Request q = i == 0 ? first : request_of(a, i * NT + tid);
    const uint32_t ends = block_scan(q.have > q.need ? q.have - q.need : 0, c.part, tid);
    if (tid == NT - 1) s_total = ends;
    __syncthreads();
    back += s_total;
  }
  const int64_t top = before + back;
  if (before < 0 || top > a.capacity) return;  // no such stack
  // page f that comes back, counted over the batch, lies f below the top
  int64_t done = 0;
  for (int i = 0; back > 0 && i < chunks; ++i) {
    const Request q = i == 0 ? first : request_of(a, i * NT + tid);
    const uint32_t n = q.have > q.need ? q.have - q.need : 0;
    const uint32_t ends = block_scan(n, c.part, tid);
    c.slot[tid] = static_cast<int32_t>(q.slot);
    c.from[tid] = q.need;
    c.ends[tid] = ends;
    __syncthreads();
    const uint32_t all = c.ends[NT - 1];
    move_pages(
        c, all, tid, [&](uint32_t, int r, int i) { return a.block_table[c.slot[r] * a.stride_table + c.from[r] + i]; },
        [&](uint32_t f, int, int, int32_t page) { a.free_pages[top - 1 - (done + f)] = page; });
    if (n > 0) a.num_pages[q.slot] = q.need;
    done += all;
    __syncthreads();
  }
  // the stack is whole (the barrier above orders its stores for this workgroup); now it is taken from
  __syncthreads();
  int64_t taken = 0, wanted = 0;
  for (int i = 0; i < chunks; ++i) {  // (a request that gave pages back needs none)
    const Request q = i == 0 ? first : request_of(a, i * NT + tid);
    const uint32_t n = q.need > q.have ? q.need - q.have : 0;
    const uint32_t ends = block_scan(n, c.part, tid);
    const bool served = n > 0 && wanted + ends <= top;
    c.slot[tid] = served ? static_cast<int32_t>(q.slot) : -1;
    c.from[tid] = q.have;
    c.ends[tid] = ends;
    __syncthreads();
    const uint32_t all = c.ends[NT - 1];
    move_pages(
        c, all, tid, [&](uint32_t f, int r, int) { return c.slot[r] < 0 ? 0 : a.free_pages[top - 1 - (wanted + f)]; },
        [&](uint32_t, int r, int i, int32_t page) {
          if (c.slot[r] >= 0) a.block_table[c.slot[r] * a.stride_table + c.from[r] + i] = page;
        });
    if (served) a.num_pages[q.slot] = q.need;
    if (tid == 0) s_served = 0;
    __syncthreads();
    if (served) atomicMax(&s_served, ends);
    __syncthreads();
    if (s_served > 0) taken = wanted + s_served;
    wanted += all;
    __syncthreads();
  }
  if (tid == 0) *a.num_free = static_cast<int32_t>(top - taken);
}

constexpr int kMapThreads = 256;

__global__ __launch_bounds__(kMapThreads) void slot_maps_kernel(const eagle4_slot_maps_args a) {
  const int r = blockIdx.x, tid = threadIdx.x + blockIdx.y * kMapThreads, step = kMapThreads * gridDim.y;
  int64_t end = 0;
  if (r < a.num_reqs) {
    const int64_t slot = e4::ld(a.idx_mapping, r), context = e4::ld(a.context_lens, r);
    const int64_t start = e4::ld(a.query_start_loc, r);
    end = e4::ld(a.query_start_loc, r + 1);
    const bool known = slot >= 0 && slot < a.state_slots;
    int held = known ? a.num_pages[slot] : 0;
    held = held < a.max_pages ? held : a.max_pages;
    const int32_t* const table = a.block_table + (known ? slot : 0) * a.stride_table;
    const int64_t last = end < a.rows ? end : a.rows;
    if (r == 0)  // rows before the first request's
      for (int64_t row = tid; row < start && row < a.rows; row += step) a.slots[row] = -1;
    const uint32_t page = static_cast<uint32_t>(a.page);
    for (int64_t row = (start > 0 ? start : 0) + tid; row < last; row += step) {
      const int64_t position = context + (row - start);
      int64_t at = -1;
      if (position >= 0 && position < static_cast<int64_t>(held) * page) {  // (a product below 2^31 is taken apart in 32 bits)
        int64_t entry;
        if (position < (int64_t{1} << 31))
          entry = static_cast<uint32_t>(position) / page;
        else
          entry = position / page;
        at = static_cast<int64_t>(table[entry]) * page + (position - entry * page);
      }
      a.slots[row] = at;
    }
    if (a.batch_table != nullptr)
      for (int i = tid; i < a.max_pages; i += step) a.batch_table[r * a.stride_batch + i] = i < held ? table[i] : 0;
  }
  if (r + 1 >= a.num_reqs)  // rows behind the last request's
    for (int64_t row = (end > 0 ? end : 0) + tid; row < a.rows; row += step) a.slots[row] = -1;
}

bool tab_ok(const eagle4_itab& t) { return t.ptr != nullptr && e4::is_index_dtype(t.dtype); }

}  // namespace

extern "C" int eagle4_resize_tables(const eagle4_resize_tables_args* a, void* stream) {
  if (a->num_reqs == 0) return EAGLE4_OK;
  if (a->num_reqs < 0 || a->num_reqs > (1 << 20) || a->slots < 1 || a->max_pages < 1 || a->max_pages > (1 << 21) || a->page < 1 ||
      a->capacity < 0 || a->capacity > INT32_MAX || a->block_table == nullptr || a->num_pages == nullptr ||
      (a->free_pages == nullptr && a->capacity > 0) || a->num_free == nullptr || !tab_ok(a->idx_mapping) || !tab_ok(a->lens) ||
      a->stride_table < (a->slots > 1 ? a->max_pages : 0))
    return EAGLE4_NOT_COVERED;
  resize_tables_kernel<<<1, NT, 0, static_cast<hipStream_t>(stream)>>>(*a);
  return E4_LAUNCH_STATUS();
}

extern "C" int eagle4_slot_maps(const eagle4_slot_maps_args* a, void* stream) {
  if (a->rows == 0 && a->num_reqs == 0) return EAGLE4_OK;
  if (a->rows < 0 || a->num_reqs < 0 || a->num_reqs > (1 << 20) || (a->rows > 0 && a->slots == nullptr) || a->page < 1 ||
      (a->num_reqs > 0 &&
       (a->state_slots < 1 || a->max_pages < 1 || a->max_pages > (1 << 21) || a->block_table == nullptr || a->num_pages == nullptr ||
        !tab_ok(a->idx_mapping) || !tab_ok(a->context_lens) || !tab_ok(a->query_start_loc) ||
        a->stride_table < (a->state_slots > 1 ? a->max_pages : 0) ||
        (a->batch_table != nullptr && a->num_reqs > 1 && a->stride_batch < a->max_pages))))
    return EAGLE4_NOT_COVERED;
  const int requests = a->num_reqs > 0 ? a->num_reqs : 1;
  // about four rows (or table entries) a thread, over all requests alike
  const int64_t each = (a->rows + requests - 1) / requests;
  const int64_t most = each > a->max_pages ? each : a->max_pages;
  int shares = static_cast<int>((most + 4 * kMapThreads - 1) / (4 * kMapThreads));
  shares = shares < 1 ? 1 : shares > 64 ? 64 : shares;
  slot_maps_kernel<<<dim3(requests, shares), kMapThreads, 0, static_cast<hipStream_t>(stream)>>>(*a);
  return E4_LAUNCH_STATUS();
}
