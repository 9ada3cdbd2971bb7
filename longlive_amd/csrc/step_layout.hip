// Layout of a step of several streams on the device (ll_step_layout): from the new tokens and the keys of every stream, where its rows
// begin, what each token's position and row of the paged cache are, and which free pages go to whom.
//
//   start[b] = n[0] + .. + n[b - 1],  want[b] = ceil((m[b] + n[b]) / P) - ceil(m[b] / P),  first[b] = want[0] + .. + want[b - 1]
//
// for n new tokens and m keys held.  A workgroup takes 1024 streams at a time, one a thread: two prefix sums, over tokens and, with the tokens
// that have a row at all, over pages, each in the wave by moves between lanes and across waves through LDS.  The tokens of these streams
// then find theirs in LDS, a search of ten steps, and work out key, page and row by themselves: a page is new where its number is no smaller
// than ceil(m / P), and then comes from the list of free ones, so no token waits for what another one writes into the table.
//
// With more tokens than a workgroup's share, every workgroup forms the sums of all streams up to its tokens, the first one writes what
// belongs to streams, and nothing passes between workgroups.  Lengths that the launch replaces (kv_lens_out is kv_lens, or a cursor)
// are then copied aside first, by a launch of its own, since workgroups that begin late still read them.
//
// What bounds it: the launch and one chain of dependent reads (lengths, sums, table, free pages), next to which the bytes are nothing.  From call to call,
// and on the device by a kernel trace, which lengthens what is as short: 24 streams of one token 5.6 to 6.4 us and 2.7 to 3.0, where a fill of one number takes
// 3.5 from call to call; 1000 streams of 1 to 4 tokens 6.3 to 6.6 and 6.0 to 6.3; 100 prompts of 50 to 4096 tokens 5.9 to 6.3 and 5.2 to 5.9.
#include "ll_common.h"

#include <algorithm>
#include <utility>

namespace ll {

constexpr int kLayoutThreads = 1024;
// Of a workgroup, where there are several: us of the 100 prompts by 1024 6.3, 2048 6.2, 4096 7.5, 8192 11.4.
constexpr uint32_t kLayoutTokens = 2048;
// Streams and tokens up to which a workgroup of so many threads does: us with 256 / with 1024: 24 streams of one token 2.74 / 3.06, 256 of 4 5.9 / 3.8,
// 64 of 30 8.4 / 4.5.
constexpr int kLayoutFew = 256;

struct LayoutParams {
  const int32_t *new_lens, *kv_lens, *cursor_from;
  int32_t *q_starts, *kv_out, *cursor, *wanted;
  int32_t* table;
  int64_t table_stride;
  uint32_t width;
  Divisor page;
  const int32_t* free_pages;
  uint32_t n_free;
  const int32_t *group_starts, *prefix_lens;
  int groups, streams;
  uint32_t tokens, per_workgroup;
  int64_t *positions, *slots;
};

// The sum over this lane and those before it, no more than `most`, which is below 2^31 as every addend is.
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v, uint32_t most) {
#define LL_DPP_ADD(ctrl, row_mask) v = min(v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, row_mask, 0xF, true), most)
  LL_DPP_ADD(0x111, 0xF);  // row_shr:1, 2, 4, 8
  LL_DPP_ADD(0x112, 0xF);
  LL_DPP_ADD(0x114, 0xF);
  LL_DPP_ADD(0x118, 0xF);
  LL_DPP_ADD(0x142, 0xA);  // row_bcast:15 into rows 1 and 3
  LL_DPP_ADD(0x143, 0xC);  // row_bcast:31 into rows 2 and 3
#undef LL_DPP_ADD
  return v;
}

// The sum over the threads before this one, and `total`, over all of them; both no more than `most`.  of_waves: a word for each wave.
template <int THREADS>
__device__ __forceinline__ uint32_t threads_before(uint32_t v, uint32_t most, uint32_t* of_waves, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t upto = lanes_upto(v, most);
  uint32_t before = (uint32_t)__shfl_up((int)upto, 1);
  if (lane == 0) before = 0;
  if (lane == 63) of_waves[wave] = upto;
  __syncthreads();
  const uint32_t waves = lanes_upto(lane < THREADS / 64 ? of_waves[lane] : 0, most);
  total = (uint32_t)__builtin_amdgcn_readlane((int)waves, 63);
  const uint32_t ahead = (uint32_t)__shfl((int)waves, max(wave - 1, 0));
  return min(before + (wave ? ahead : 0), most);
}

// Ahead of a launch of several workgroups that replaces what it reads: the lengths and the cursor as they are.
__global__ __launch_bounds__(256) void layout_keep_kernel(const int32_t* kv_lens, int streams, const int32_t* cursor, int32_t* kept) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < streams) kept[i] = kv_lens[i];
  if (i == streams) kept[i] = cursor ? *cursor : 0;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void step_layout_kernel(LayoutParams p) {
  __shared__ uint32_t of_waves[2][THREADS / 64];
  __shared__ int starts[THREADS], held[THREADS], first_page[THREADS], ahead[THREADS];
  const int tid = threadIdx.x;
  const bool writes_streams = blockIdx.x == 0;
  const uint32_t t0 = blockIdx.x * p.per_workgroup, t1 = (uint32_t)min((uint64_t)t0 + p.per_workgroup, (uint64_t)p.tokens);
  const uint32_t taken = p.cursor_from ? (uint32_t)max(*p.cursor_from, 0) : 0;
  uint32_t start = 0, pages = 0;  // of the streams before
  for (int b0 = 0; b0 < p.streams; b0 += THREADS) {
    const int b = b0 + tid, count = min(THREADS, p.streams - b0);
    uint32_t n = 0, m = 0;
    if (b < p.streams) {
      m = (uint32_t)max(p.kv_lens[b], 0);
      n = min((uint32_t)max(p.new_lens[b], 0), 0x7fffffffu - m);
      n = min(n, p.tokens);
    }
    uint32_t all;
    const uint32_t mine = min(start + threads_before<THREADS>(n, p.tokens, of_waves[0], all), p.tokens);
    n = min(n, p.tokens - mine);  // tokens that have no row are not laid out
    const uint32_t have = min((m + p.page.d - 1) / p.page, p.width), need = min((m + n + p.page.d - 1) / p.page, p.width);
    uint32_t all_pages;
    const uint32_t first = pages + threads_before<THREADS>(need - have, 0x7fffffffu, of_waves[1], all_pages);
    if (b < p.streams) {
      int shared = 0;
      if (p.groups > 0) {
        int g = 0;  // the last group that begins at or before the stream
        if (p.group_starts) {
          int end = p.groups + 1;
          while (end - g > 1) {
            const int at = (g + end) >> 1;
            if (p.group_starts[at] <= b) g = at;
            else end = at;
          }
          if (p.group_starts[g] > b) g = p.groups;
        }
        shared = g < p.groups ? max(p.prefix_lens[g], 0) : 0;
      }
      starts[tid] = (int)mine;
      held[tid] = (int)m;
      first_page[tid] = (int)(first - have);
      ahead[tid] = shared;
      if (writes_streams) {
        p.q_starts[b] = (int)mine;
        p.kv_out[b] = (int)(m + n);
      }
    }
    const uint32_t end = min(start + all, p.tokens);
    __syncthreads();
    for (uint32_t t = max(t0, start) + tid; t < min(t1, end); t += THREADS) {
      int at = 0, stop = count;  // the last stream that begins at or before the token
      while (stop - at > 1) {
        const int mid = (at + stop) >> 1;
        if (starts[mid] <= (int)t) at = mid;
        else stop = mid;
      }
      const uint32_t key = (uint32_t)held[at] + t - (uint32_t)starts[at];
      const uint32_t entry = key / p.page, row = key - entry * p.page.d;
      int page = -1;
      if (entry < p.width) {
        int32_t* const in_table = p.table + (int64_t)(b0 + at) * p.table_stride + entry;
        const uint32_t have = ((uint32_t)held[at] + p.page.d - 1) / p.page;
        if (entry >= have) {
          const uint64_t next = (uint64_t)taken + (uint32_t)(first_page[at] + (int)entry);
          if (next < p.n_free) page = p.free_pages[next];
          if (row == 0) *in_table = page;
        } else {
          page = *in_table;
        }
      }
      p.positions[t] = (int64_t)ahead[at] + key;
      p.slots[t] = page >= 0 ? (int64_t)page * p.page.d + row : -1;
    }
    start = end;
    pages += all_pages;
    if (!writes_streams && start >= t1) return;
    __syncthreads();  // before the next streams take the places of these
  }
  for (uint32_t t = max(t0, start) + tid; t < t1; t += THREADS) {  // rows behind the last stream
    p.positions[t] = 0;
    p.slots[t] = -1;
  }
  if (writes_streams && tid == 0) {
    p.q_starts[p.streams] = (int)start;
    *p.wanted = (int)pages;
    if (p.cursor) *p.cursor = (int)min((uint64_t)taken + pages, (uint64_t)max(p.n_free, taken));
  }
}

static bool layout_in_parts(const ll_step_layout_args& a) { return a.tokens > kLayoutTokens; }
// Whether several workgroups would read what one of them replaces.
static bool layout_keeps(const ll_step_layout_args& a) { return layout_in_parts(a) && a.streams > 0 && (a.kv_lens_out == a.kv_lens || a.cursor); }

// Whether two ranges of bytes share one.
static bool meet(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t at = (uintptr_t)a, bt = (uintptr_t)b;
  return a_bytes > 0 && b_bytes > 0 && (at < bt ? bt - at < (uint64_t)a_bytes : at - bt < (uint64_t)b_bytes);
}
// Whether a range of bytes shares one with the table's rows; it may lie between them.
static bool meets_table(const ll_step_layout_args& a, const void* b, int64_t bytes) {
  const int64_t width = a.table_width * 4, stride = (a.table_stride < 0 ? -a.table_stride : a.table_stride) * 4;
  if (bytes <= 0 || width == 0 || a.streams == 0) return false;
  const int32_t* const low = a.table_stride < 0 ? a.page_table + (a.streams - 1) * a.table_stride : a.page_table;
  const int64_t off = (int64_t)((uintptr_t)b - (uintptr_t)low);
  if (off < width) return off + bytes > 0;
  if (a.streams == 1) return false;
  const int64_t row = off / stride, in_row = off - row * stride;
  return row < a.streams && (in_row < width || (row + 1 < a.streams && in_row + bytes > stride));
}

// What is written lies in places of its own: with several workgroups the first replaces what later ones would still read.
static int check_apart(const ll_step_layout_args& a) {
  const auto list = [](const void* at, int64_t bytes) { return std::pair<const void*, int64_t>(at, at ? bytes : 0); };
  const auto inputs = {list(a.new_lens, 4 * a.streams), list(a.kv_lens, 4 * a.streams), list(a.free_pages, 4 * a.n_free),
                       list(a.group_starts, a.groups ? 4 * (a.groups + 1) : 0), list(a.prefix_lens, 4 * a.groups)};
  const std::pair<const void*, int64_t> outputs[] = {list(a.kv_lens_out, 4 * a.streams),   list(a.cursor, 4),          list(a.q_starts, 4 * (a.streams + 1)),
                                                     list(a.positions, 8 * a.tokens),      list(a.slots, 8 * a.tokens), list(a.pages_wanted, 4),
                                                     list(a.workspace, layout_keeps(a) ? 4 * (a.streams + 1) : 0)};
  LL_REQUIRE(a.streams <= 1 || a.table_width == 0 || a.table_stride >= a.table_width || -a.table_stride >= a.table_width,
             "ll_step_layout: rows of the page table overlap, %lld apart for %lld entries", (long long)a.table_stride, (long long)a.table_width);
  bool apart = true;
  for (const auto& in : inputs) {
    apart = apart && !meets_table(a, in.first, in.second);
    for (const auto& out : outputs) {
      const bool in_place = out.first == a.kv_lens_out && in.first == a.kv_lens && out.first == in.first;
      apart = apart && (in_place || !meet(in.first, in.second, out.first, out.second));
    }
  }
  for (const auto& out : outputs) {
    apart = apart && !meets_table(a, out.first, out.second);
    for (const auto* other = outputs; other < &out; ++other) apart = apart && !meet(other->first, other->second, out.first, out.second);
  }
  LL_REQUIRE(apart, "ll_step_layout: outputs (page table, cursor, new lengths, results) overlap inputs or one another; only the new lengths may replace the held ones");
  return LL_OK;
}

static int check_layout(const ll_step_layout_args* a) {
  LL_REQUIRE(a, "ll_step_layout: no arguments");
  // as many as attention takes: the kernel counts streams on by a workgroup's threads, and adds two groups' numbers, in 31 bits
  LL_REQUIRE(a->streams >= 0 && a->streams <= 0xfffffff, "ll_step_layout: %lld streams", (long long)a->streams);
  LL_REQUIRE(a->tokens >= 0 && a->tokens <= 0x7fffffffll, "ll_step_layout: %lld tokens", (long long)a->tokens);
  LL_REQUIRE(a->page_size > 0, "ll_step_layout: pages of %d rows", a->page_size);
  LL_REQUIRE(a->table_width >= 0 && a->table_width <= 0x7fffffffll, "ll_step_layout: a table of %lld pages a stream", (long long)a->table_width);
  LL_REQUIRE(a->n_free >= 0 && a->n_free <= 0x7fffffffll, "ll_step_layout: %lld free pages", (long long)a->n_free);
  LL_REQUIRE(a->groups >= 0 && a->groups <= 0xfffffff, "ll_step_layout: %lld groups", (long long)a->groups);
  return LL_OK;
}

}  // namespace ll

extern "C" int ll_step_layout_workspace(const ll_step_layout_args* a, size_t* bytes) {
  using namespace ll;
  if (int rc = check_layout(a)) return rc;
  LL_REQUIRE(bytes, "ll_step_layout_workspace: nowhere to put the answer");
  *bytes = layout_keeps(*a) ? ((size_t)a->streams + 1) * sizeof(int32_t) : 0;
  return LL_OK;
}

extern "C" int ll_step_layout(const ll_step_layout_args* a, void* stream) {
  using namespace ll;
  if (int rc = check_layout(a)) return rc;
  LL_REQUIRE(a->q_starts && a->pages_wanted, "ll_step_layout: null starts or pages wanted");
  LL_REQUIRE(a->streams == 0 || (a->new_lens && a->kv_lens && a->kv_lens_out), "ll_step_layout: null lengths");
  LL_REQUIRE(a->tokens == 0 || (a->positions && a->slots), "ll_step_layout: null positions or slots");
  LL_REQUIRE(a->streams == 0 || a->table_width == 0 || a->page_table, "ll_step_layout: null page table");
  LL_REQUIRE(a->n_free == 0 || a->free_pages, "ll_step_layout: null list of free pages");
  LL_REQUIRE(a->groups == 0 || a->prefix_lens, "ll_step_layout: groups without lengths of what they share");
  LL_REQUIRE(a->groups <= 1 || a->group_starts, "ll_step_layout: %lld groups without their beginnings", (long long)a->groups);
  if (int rc = check_apart(*a)) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  LayoutParams p{};
  p.new_lens = a->new_lens;
  p.kv_lens = a->kv_lens;
  p.cursor_from = a->cursor;
  p.q_starts = a->q_starts;
  p.kv_out = a->kv_lens_out;
  p.cursor = a->cursor;
  p.wanted = a->pages_wanted;
  p.table = a->page_table;
  p.table_stride = a->table_stride;
  p.width = (uint32_t)a->table_width;
  p.page = divisor((uint32_t)a->page_size);
  p.free_pages = a->free_pages;
  p.n_free = (uint32_t)a->n_free;
  p.group_starts = a->group_starts;
  p.prefix_lens = a->prefix_lens;
  p.groups = (int)a->groups;
  p.streams = (int)a->streams;
  p.tokens = (uint32_t)a->tokens;
  p.positions = a->positions;
  p.slots = a->slots;
  const bool parts = layout_in_parts(*a);
  p.per_workgroup = parts ? kLayoutTokens : (uint32_t)a->tokens;
  if (layout_keeps(*a)) {
    LL_REQUIRE(a->workspace && (uintptr_t)a->workspace % 4 == 0 && a->workspace_bytes >= ((size_t)a->streams + 1) * sizeof(int32_t),
               "ll_step_layout: a workspace of %zu bytes is needed", ((size_t)a->streams + 1) * sizeof(int32_t));
    int32_t* kept = static_cast<int32_t*>(a->workspace);
    layout_keep_kernel<<<(uint32_t)(a->streams / 256 + 1), 256, 0, s>>>(a->kv_lens, p.streams, a->cursor, kept);
    LL_CHECK_LAUNCH("ll_step_layout");
    p.kv_lens = kept;
    p.cursor_from = kept + a->streams;
  }
  const uint32_t grid = parts ? (uint32_t)((a->tokens + kLayoutTokens - 1) / kLayoutTokens) : 1;
  if (a->streams <= kLayoutFew && a->tokens <= kLayoutFew)
    step_layout_kernel<kLayoutFew><<<grid, kLayoutFew, 0, s>>>(p);
  else
    step_layout_kernel<kLayoutThreads><<<grid, kLayoutThreads, 0, s>>>(p);
  LL_CHECK_LAUNCH("ll_step_layout");
  return LL_OK;
}
