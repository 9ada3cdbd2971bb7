// Attention of a batch of streams of different length (ll_ragged_attention): new tokens over the keys of a paged cache, or
// queries over encoder states whose number differs from stream to stream; and over beginnings that groups of streams share
// (ll_shared_prefix_attention, see "beginnings that groups attend together").
//
//   out[t, h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale * (q[t, h] . k_j - max)),   j over the keys that row t may see
//
// The rows of a kv head's queries, (token, head of the group) one behind the other, are cut into tiles of 128, and the keys of a tile
// into parts of about as many steps as the plan says; the workgroups of the launch, as many as the device holds at once, take
// these items in turn and find them by prefix sums over the streams, whose lengths only the device knows.  A workgroup of four
// waves multiplies
//   S^T = K Q^T  and  O^T = V^T P^T   (v_mfma_f32_32x32x16),
// so that a lane owns one row: its maximum and sum need one exchange between the wave's halves, its mask is a word of bits, and its
// rescaling is a multiplication by a scalar.  The probabilities leave the first product in the registers in which the second one
// wants them, keys permuted; V^T is read permuted alike by the LDS read that transposes.
//
//   * Tiles of more than 32 rows: a wave owns 32 rows, and all four walk the same keys, 64 a step, through two stages in LDS, scores a
//     step ahead of probabilities: under the 16 products of S^T of the next step and the 16 of O^T of this one run this step's
//     exponentials and the next one's maximum.
//   * Tiles of up to 32 rows (single tokens, drafts): all waves own the same rows, and each walks every fourth group of 32 keys
//     with LDS of its own and no barrier, K of the next group on its way from the moment the scores are done, V from the moment
//     they are used; the four results are merged at the end.
//   * The results of a tile's parts go to memory as they are, and a second launch joins them in order.
//
// K and V go straight from memory to LDS, 1024 bytes a load.  Where the rows lie is looked up one step ahead, an entry of the
// page table per lane, also straight to LDS, so that no register load stands between the loads under way and their wait.
//
// What bounds it (bf16, 128 columns; the card's own copy of 2 GiB runs at 4.9 TB/s, the library's 8192^3 product at 1219 TFLOP/s):
// single tokens of 32 streams over 500 to 16384 keys take 102 to 108 us, 4.6 to 4.9 TB/s of K and V; 2640 x 24 heads over 13200 keys
// take 424 to 442 us, 0.97 to 1.0 PFLOP/s, where the matrix unit is busy for half of the cycles, 6.1 other vector instructions go with each
// of its instructions and the clock is down at 2.0 GHz.  Over the same keys as rows one behind the other it is 388, next to 380 of the dense
// kernel (ll_attention_bf16): a tenth goes into where pages lie.  With fewer steps per item its beginning shows (places, then keys, then
// the first scores, one behind the other, some 5 us beside the other workgroup of the unit): 532 x 40 / 8 heads over 9000 keys 118 us, 0.81
// PFLOP/s, 3 x 2640 x 24 over 60 to 512 encoder states 43 us, 0.56 PFLOP/s.
// Registers: with 64 columns three workgroups of a unit leave 168 a lane, of which 4 to 8 more would be needed (20 to 36 bytes of scratch
// memory); with 128 columns 230 to 246 and none.  41 to 82 scalars are kept in lanes of vector registers.  With shared beginnings 168 and 68 to 76
// bytes, 250 to 254 and none, 62 to 111 scalars.
#include "ll_types16.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

namespace ll {

constexpr int kRaThreads = 256;
constexpr int kRaTileRows = 128;  // rows of a workgroup, 32 a wave
constexpr int kRaKeys = 64;       // keys of a step
constexpr int kRaClearGroups = 16;
constexpr uint32_t kRaLeastWideSteps = 10;  // of a part, where tiles are not alike
constexpr float kLog2E = 1.4426950408889634f;
// Of the joining launch, times two passes over a tile's rows: 17 streams over 100 to 2400 masked states 59.6 us, with 512 and four 61.0, with
// 512 and one 64.9.
constexpr uint32_t kRaJoinGroups = 256;

// Where keys lie: in the pages of a table, in rows one behind the other, in such rows with a mask.
// With shared beginnings: in the pages of a table, behind those of the beginning of the stream's group.  Listed: a launch ahead has listed the
// items, beginnings of whole groups among them.
constexpr int kRaPaged = 0, kRaRows = 1, kRaMaskedRows = 2, kRaPrefixed = 3, kRaListed = 4;

// An item of every kv head, as listed ahead.
struct RaListedItem {
  int q0, rows, first, len, base, prefix_len, prefix_row, table_row, s_begin, s_end;
  int slot;  // of the part's results, -1: they are the tile's
  int unused;  // to whole 16 bytes
};
struct RaList {
  uint32_t prefix_items, single_items, items;  // items of beginnings; with those that take a workgroup; with those that take a wave
  uint32_t wide_part, narrow_part;             // steps of a part of a stream's own keys, for more than 32 rows and for fewer
};
struct RaJoined {  // of a stream: parts of its group's beginning, or steps of it ahead of its own
  int parts, ahead, joined;
};

struct RaParams {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_stride_token, q_stride_head, out_stride_token, out_stride_head;
  int64_t n_queries;
  int streams;
  const int32_t* q_starts;
  const uint16_t *k, *v;
  int64_t k_stride_head, v_stride_head;
  uint32_t k_stride_page, k_stride_row, v_stride_page, v_stride_row;
  const int32_t* page_table;
  int64_t table_stride;
  int64_t table_keys;  // keys that a stream's row of the table reaches
  uint32_t n_pages;
  Divisor page;
  const int32_t *kv_lens, *k_starts, *k_lens;
  const uint8_t* key_mask;
  int64_t n_keys;
  float scale_log2;
  int causal;
  int heads, kv_heads;
  Divisor group;          // heads of a kv head
  uint32_t window, sink;  // window 0: none
  uint32_t groups;        // workgroups that take the items
  // Steps of a part, for tiles of more rows and for streams of up to 32 rows.  0 records: nothing is cut.
  uint32_t part_steps, narrow_part_steps;
  float part_share;       // not 0: part_steps follow from the streams, this times the steps of all wide tiles of a head
  uint32_t records;       // of a kv head, 32 rows each
  float* record_mem;      // [kv head][records]: 32 x D columns, then reference point and sum of each row
  // Shared beginnings.
  const int32_t *group_starts, *prefix_lens, *prefix_table;
  int64_t prefix_stride, prefix_keys;  // keys that a row of the table reaches
  int n_groups;
  // Listed: results of parts lie by row in record_mem, [prefix_parts + own_parts][n_queries][heads] of D columns, then as many reference points
  // and sums.
  uint32_t prefix_parts, own_parts;    // parts of a tile at most
  RaList* list;
  RaListedItem* listed;
  uint32_t most_listed;
  RaJoined* joined;                    // [streams]
};

// Positions of 16-byte pieces in an LDS row of D columns.  The reads of a wave then go through all banks: 8 neighbouring rows of one
// column of K, 4 rows by two columns of V.
template <int D>
__device__ __forceinline__ int k_piece(int row, int piece) {
  return D == 128 ? piece ^ (row & 15) : piece ^ ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_piece(int row, int piece) {
  return D == 128 ? piece ^ (4 * (row & 3)) ^ (2 * ((row >> 2) & 1)) : piece ^ (4 * ((row >> 1) & 1)) ^ (2 * ((row >> 2) & 1));
}

__device__ __forceinline__ float exchange_max(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float exchange_sum(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 16 or 4 bytes per lane from memory straight into LDS at lds + 16 (4) * lane.  asm statements, so that the compiler does not wait
// for them ahead of LDS reads of other data; wait_loads does.
__device__ __forceinline__ void load16_to_lds(uint32_t offset, const void* base, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
__device__ __forceinline__ void load16_to_lds(const void* from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
__device__ __forceinline__ void load4_to_lds(const void* from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
// All but the last N loads of this wave have arrived.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// This wave's LDS reads have their data: what they read may be overwritten.
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}
template <typename P>
__device__ __forceinline__ const P* uniform_pointer(const P* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const P*>((uintptr_t)(((uint64_t)hi << 32) | lo));
}

// What rows of keys that do not exist are read from.
__device__ const uint4 kRaZeros[1] = {{0, 0, 0, 0}};

__device__ __forceinline__ int64_t stream_start(const RaParams& p, int b) { return min(max((int64_t)p.q_starts[b], (int64_t)0), p.n_queries); }

// The lowest n of 64 bits, for any n.
__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : ~(~0ull << n); }

// A group of streams, its rows of q and the keys that it shares.
struct RaGroup {
  int q0, n, len;
  bool joined;  // its rows attend the beginning together, each stream's rows then its own keys, and the two are joined; else one behind the other
};
// Going together saves a group of m streams about m / 2 tiles of every step of the beginning, what its streams' last tiles lack, and costs two
// records of every row: it is done from this many steps times streams to a tile on.  us with all groups together / with those that gain: 16 groups
// of 4 streams x 33 to 64 tokens x 32 / 8 heads of 128 columns over 2000 shared keys 226 / 173 (none gains), 4 of 16 over 1000 143 / 111, 16 of 4
// x 12 of 64 over 2000 76 / 76 (all do), one of 16 x 16 / 4 of 64 over 2000 36 / 43.
constexpr int kRaJoinedCost = 28;
__device__ __forceinline__ int group_len(const RaParams& p, int g) { return (int)min((int64_t)max(p.prefix_lens[g], 0), p.prefix_keys); }
__device__ __forceinline__ RaGroup group_of(const RaParams& p, int g) {
  const int from = p.group_starts ? min(max(p.group_starts[g], 0), p.streams) : 0;
  const int to = p.group_starts ? min(max(p.group_starts[g + 1], from), p.streams) : p.streams;
  RaGroup r;
  const int limit = (int)p.n_queries;
  r.q0 = min(max(p.q_starts[from], 0), limit);
  r.n = max(min(max(p.q_starts[to], 0), limit) - r.q0, 0);
  r.len = group_len(p, g);
  r.joined = p.prefix_parts > 0 && to - from > 1 && r.n > 0 &&
             (int64_t)(to - from) * (r.len / kRaKeys) >= (int64_t)kRaJoinedCost * (((uint32_t)r.n * p.group.d + kRaTileRows - 1) / kRaTileRows);
  return r;
}
// The group of a stream, -1 for none.
__device__ __forceinline__ int group_of_stream(const RaParams& p, int b) {
  if (p.n_groups == 0) return -1;
  if (!p.group_starts) return 0;
  int g = 0, end = p.n_groups + 1;  // the last that begins at or before it
  while (end - g > 1) {
    const int at = (g + end) >> 1;
    if (p.group_starts[at] <= b) g = at;
    else end = at;
  }
  return g < p.n_groups && p.group_starts[g] <= b ? g : -1;
}
__device__ __forceinline__ int steps_of(int keys) { return (keys + kRaKeys - 1) / kRaKeys; }
// Parts of a tile that takes so many steps, no more than `most`.
__device__ __forceinline__ int shared_parts(uint32_t steps, uint32_t per_part, uint32_t most) { return (int)min((steps + per_part - 1) / per_part, most); }

// What a workgroup does next: a part of a tile.
struct RaItem {
  int64_t q0;               // first row of q of the stream
  int rows, first;          // rows of the stream (token, head of the group), the tile's first
  int len;                  // keys of the stream that there is a place for
  int base;                 // paged: the position of its first token
  int key0;                 // rows of keys: row of key 0
  const int32_t* pages;     // paged: the stream's row of the table
  int sink_steps, from_step;  // the tile's steps: 0 .. sink_steps - 1, and then from from_step on
  int s_begin, s_end;       // of these, the part's
  int n_parts, part;
  uint32_t record;          // of part 0; the others follow, each as many records as the tile has groups of 32 rows
  // With shared beginnings: of the tile's steps the first go over the beginning, whose keys have the numbers -64 prefix_steps and up.
  const int32_t* prefix_pages;
  int prefix_steps, prefix_len;
  int slot;                 // where the part's results go, to be joined with others; -1: they are the tile's
};

// The streams b0 .. b0 + 63, one a lane.
struct RaStreams {
  int q0, n, len, base, key0;
  int parts;                          // at most: of the tile that sees most keys
  uint32_t items_upto, records_upto;  // of these and the streams before
  int shares, prefix_len;             // with shared beginnings: the group, its keys
};

// Steps of a tile whose first and last token sit at pos0 and pos1, of a stream of len keys.
struct RaSpan {
  int sink_steps, from_step, n_steps;
};
__device__ __forceinline__ RaSpan span_of(const RaParams& p, int len, int pos0, int pos1) {
  const int end = p.causal ? min(pos1 + 1, len) : len;
  const int from = p.window && pos0 >= (int)p.window ? pos0 - (int)p.window + 1 : 0;
  const int end_step = end > 0 ? (end - 1) / kRaKeys + 1 : 0;
  RaSpan s;
  s.from_step = from / kRaKeys;
  s.sink_steps = min((int)(((int64_t)min((int)p.sink, from) + kRaKeys - 1) / kRaKeys), s.from_step);
  s.n_steps = min(s.sink_steps, end_step) + max(end_step - s.from_step, 0);
  return s;
}
// Tiles of a stream's rows.
__device__ __forceinline__ int tiles_of(int rows) { return rows > 0 ? (rows - 1) / kRaTileRows + 1 : 0; }
// Records of a tile's part.
__device__ __forceinline__ int record_groups(int rows) { return rows <= 32 ? 1 : kRaTileRows / 32; }

// The sum over this lane and those before it, by moves between the lanes of a row of 16 and then from row to row.
#define LL_DPP_ADD(v, ctrl, row_mask) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, row_mask, 0xF, true)
__device__ __forceinline__ uint32_t sum_upto(uint32_t v) {
  LL_DPP_ADD(v, 0x111, 0xF);  // row_shr:1
  LL_DPP_ADD(v, 0x112, 0xF);  // row_shr:2
  LL_DPP_ADD(v, 0x114, 0xF);  // row_shr:4
  LL_DPP_ADD(v, 0x118, 0xF);  // row_shr:8
  LL_DPP_ADD(v, 0x142, 0xA);  // row_bcast:15 into rows 1 and 3
  LL_DPP_ADD(v, 0x143, 0xC);  // row_bcast:31 into rows 2 and 3
  return v;
}
#undef LL_DPP_ADD

// What is known of 64 streams, loaded at once; `items` and `records`: of the streams before.  A stream whose records would go beyond
// what there is stays whole.  COUNT_TILES: the items are the tiles that were cut.
template <int KIND, bool COUNT_TILES>
__device__ __forceinline__ RaStreams load_streams(const RaParams& p, int b0, uint32_t items, uint32_t records, uint32_t& part_steps) {
  const int lane = threadIdx.x & 63, b = min(b0 + lane, p.streams - 1);
  const int start = p.q_starts[b], next = p.q_starts[b + 1];
  const int limit = (int)p.n_queries;
  RaStreams s;
  s.q0 = min(max(start, 0), limit);
  s.n = b0 + lane < p.streams ? max(min(max(next, 0), limit) - s.q0, 0) : 0;
  s.base = 0;
  int64_t key0 = 0, len;
  s.shares = s.prefix_len = 0;
  if constexpr (KIND == kRaPaged || KIND == kRaPrefixed) {
    // positions count from the stream's last token, wherever the table and the rows of q end
    const int64_t given = max((int64_t)p.kv_lens[b], (int64_t)0);
    len = min(given, p.table_keys);
    s.base = (int)(given - ((int64_t)next - s.q0));
  } else {
    const int64_t first = p.k_starts[b], given = p.k_lens ? p.k_lens[b] : p.k_starts[b + 1];
    key0 = min(max(first, (int64_t)0), p.n_keys);
    len = min(max(p.k_lens ? given : given - key0, (int64_t)0), p.n_keys - key0);
  }
  s.len = (int)len;
  s.key0 = (int)key0;
  if constexpr (KIND == kRaPrefixed) {
    const int g = group_of_stream(p, b);
    s.prefix_len = g < 0 ? 0 : group_len(p, g);
    s.shares = max(g, 0);
  }
  const int rows = s.n * (int)p.group.d;
  const int tiles = tiles_of(rows);
  s.parts = 1;
  s.records_upto = 0;
  if (p.records) {
    uint32_t mine = 0;
    int steps = 0;
    if (tiles) {
      // Where there is a window, the first tile that sees the stream's last key sees most: up to a tile's tokens more than it, and without
      // causal order, where every tile sees that key, as many more as there are tokens (for several streams: see plan_ragged).
      const int pos1 = max(s.len - 1, s.base);
      const int pos0 = p.causal || p.streams > 1 ? pos1 - min(s.n - 1, (int)((uint32_t)(kRaTileRows - 1) / p.group) + 1) : s.base;
      steps = p.window ? span_of(p, s.len, pos0, pos1).n_steps + 1 : (s.len + kRaKeys - 1) / kRaKeys;
      if constexpr (KIND == kRaPrefixed) steps += steps_of(s.prefix_len);
    }
    if (p.part_share != 0.0f) {  // up to 64 streams, which are all here
      const int mean = p.causal && !p.window ? max(steps - s.n / (2 * kRaKeys), 1) : steps;
      const uint32_t of_tiles = rows > 32 ? (uint32_t)min((int64_t)tiles * mean, (int64_t)1 << 25) : 0;
      const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)sum_upto(of_tiles), 63);
      part_steps = max((uint32_t)__builtin_amdgcn_readfirstlane((int)fminf((float)all * p.part_share, 1e9f)), kRaLeastWideSteps);
    }
    if (tiles) {
      const uint32_t per_part = rows <= 32 ? p.narrow_part_steps : part_steps;
      s.parts = max((int)((steps + per_part - 1) / per_part), 1);
      if (s.parts > 1) mine = (uint32_t)min((int64_t)tiles * s.parts * record_groups(rows), (int64_t)p.records + 1);
    }
    // sums that do not pass 32 bits: a stream adds at most records + 1, the streams before at most as much
    s.records_upto = records + sum_upto(mine);
    if (s.records_upto > p.records) s.parts = 1;
  }
  s.items_upto = items + sum_upto(COUNT_TILES ? (s.parts > 1 ? tiles : 0) : tiles * s.parts);
  return s;
}

// Finds items one behind the other.
template <int KIND, bool COUNT_TILES>
struct RaCursor {
  int b0 = 0;
  uint32_t items = 0, records = 0;  // of the streams before b0
  uint32_t part_steps;              // of a part of a wide tile
  RaStreams s;                      // streams from b0 on
  __device__ __forceinline__ void start(const RaParams& p) {
    part_steps = p.part_steps;
    if (p.streams > 0) s = load_streams<KIND, COUNT_TILES>(p, 0, 0, 0, part_steps);
  }
  // Item `index` of a kv head, which is no smaller than the last one asked for.  All lanes call it together.  False: there are fewer.
  __device__ __forceinline__ bool find(const RaParams& p, uint32_t index, RaItem& t) {
    if (p.streams <= 0) return false;
    for (;;) {
      const uint64_t before = __builtin_amdgcn_ballot_w64(s.items_upto <= index);
      if (before != ~0ull) {
        const int at = __builtin_amdgcn_readfirstlane(__popcll(before));
        auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
        const int parts = of(s.parts);
        const uint32_t records_end = (uint32_t)of((int)s.records_upto);
        // the last tile of a stream, which sees most keys, first, and all its parts
        uint32_t left = (uint32_t)of((int)s.items_upto) - 1 - index;
        const uint32_t tile = COUNT_TILES ? left : left / (uint32_t)parts;
        t.part = COUNT_TILES ? 0 : (int)(left - tile * (uint32_t)parts);
        t.q0 = of(s.q0);
        t.rows = of(s.n) * (int)p.group.d;
        t.first = (int)tile * kRaTileRows;
        t.len = of(s.len);
        t.base = of(s.base);
        t.key0 = of(s.key0);
        t.pages = KIND == kRaPaged || KIND == kRaPrefixed ? p.page_table + (int64_t)(b0 + at) * p.table_stride : nullptr;
        const int last_row = min(t.first + kRaTileRows, t.rows) - 1;
        RaSpan span = span_of(p, t.len, t.base + (int)((uint32_t)t.first / p.group), t.base + (int)((uint32_t)last_row / p.group));
        if constexpr (KIND == kRaPrefixed) {
          t.prefix_len = of(s.prefix_len);
          t.prefix_steps = steps_of(t.prefix_len);
          t.prefix_pages = p.prefix_table + (int64_t)of(s.shares) * p.prefix_stride;
          span.n_steps += t.prefix_steps;
        }
        t.sink_steps = span.sink_steps;
        t.from_step = span.from_step;
        const uint32_t per_part = t.rows <= 32 ? p.narrow_part_steps : part_steps;
        t.n_parts = parts > 1 ? max(min((int)((span.n_steps + per_part - 1) / per_part), parts), 1) : 1;
        const int each = (span.n_steps + t.n_parts - 1) / t.n_parts;  // equal parts
        t.s_begin = min(t.part * each, span.n_steps);
        t.s_end = min(t.s_begin + each, span.n_steps);
        t.record = records_end - (uint32_t)((tiles_of(t.rows) - (int)tile) * parts * record_groups(t.rows));
        return true;
      }
      b0 += 64;
      if (b0 >= p.streams) return false;
      items = (uint32_t)__builtin_amdgcn_readlane((int)s.items_upto, 63);
      records = min((uint32_t)__builtin_amdgcn_readlane((int)s.records_upto, 63), p.records + 1);
      s = load_streams<KIND, COUNT_TILES>(p, b0, items, records, part_steps);
    }
  }
};

// Where part `part` of an item's tile has the four columns from `column` on of a row, and the row's reference point and sum.
template <int D>
__device__ __forceinline__ float* record_of(const RaParams& p, uint32_t head, const RaItem& t, int part, int row) {
  const int64_t at = (int64_t)head * p.records + t.record + (uint32_t)(part * record_groups(t.rows) + row / 32);
  return p.record_mem + at * 32 * (D + 2) + row % 32 * D;
}
template <int D>
__device__ __forceinline__ float2* record_sums(const RaParams& p, uint32_t head, const RaItem& t, int part, int row) {
  const int64_t at = (int64_t)head * p.records + t.record + (uint32_t)(part * record_groups(t.rows) + row / 32);
  return reinterpret_cast<float2*>(p.record_mem + at * 32 * (D + 2) + 32 * D) + row % 32;
}

// Listed: where part `slot` of all has a row's columns, and its reference point and sum.
template <int D>
__device__ __forceinline__ float* shared_record(const RaParams& p, uint32_t slot, int64_t token, int head) {
  return p.record_mem + (((int64_t)slot * p.n_queries + token) * p.heads + head) * D;
}
template <int D>
__device__ __forceinline__ float2* shared_sums(const RaParams& p, uint32_t slot, int64_t token, int head) {
  const int64_t rows = p.n_queries * p.heads;
  return reinterpret_cast<float2*>(p.record_mem + (int64_t)(p.prefix_parts + p.own_parts) * rows * D) + ((int64_t)slot * p.n_queries + token) * p.heads + head;
}

template <int D>
constexpr int kRaLds = 2 * 2 * kRaKeys * 2 * D + 4 * 2 * 256 + 4 * 32 * 8;  // stages, looked-up places, maxima and sums

// f(0), f(1), ... with every index a constant of its own type.
template <typename F, int... I>
__device__ __forceinline__ void each_index(F& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

// The reference point of the exponentials follows the maximum once it is 2^2 ahead: fewer rescalings, no further from 64 bits.
constexpr float kRaStep = 2.0f;
// Probabilities are exp2(score - reference + shift), so that in f16 a row's sums keep keys that are far below the largest: with none, 200000 keys
// 17.5 nats below one, half a percent of the weight, would each weigh nothing.  Sums and outputs of a row are all times 2^shift.  None where the
// reference, scaled, has no bits left for it: its rounding, the same for all keys of a row, would carry the largest beyond f16.
template <typename T>
__device__ __forceinline__ float weight_shift(float reference) {
  return T::kWeightShift != 0.0f && fabsf(reference) < 4194304.0f ? T::kWeightShift : 0.0f;
}
// Results at different reference points are joined by factors 2^((one - other) * unit): references are maxima, or with a shift the negative
// constants of the exponents.
template <typename T>
__device__ __forceinline__ float reference_unit(float scale_log2) {
  return T::kWeightShift == 0.0f ? scale_log2 : 1.0f;
}

template <typename T, int D, int KIND>
__global__ __launch_bounds__(kRaThreads, D == 64 ? 3 : 2) void ragged_attention_kernel(RaParams p) {
  constexpr int kRowBytes = 2 * D, kPieces = D / 8, kDTiles = D / 32, kSteps = D / 16;
  constexpr int kRowsPerLoad = 1024 / kRowBytes, kGroupLoads = 16 / kRowsPerLoad;  // loads of 16 rows
  constexpr int kStepBytes = kRaKeys * kRowBytes;                                  // K or V of a step
  constexpr bool kLooksUp = KIND != kRaRows, kPrefixed = KIND == kRaPrefixed || KIND == kRaListed, kPages = KIND == kRaPaged || kPrefixed;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  if (blockIdx.x >= p.groups) {  // rows outside every stream
    const int64_t first = p.streams ? stream_start(p, 0) : 0, end = p.streams ? max(stream_start(p, p.streams), first) : 0;
    const int64_t outside = first + p.n_queries - end, pieces = outside * p.heads * kPieces;
    for (int64_t i = (int64_t)(blockIdx.x - p.groups) * kRaThreads + threadIdx.x; i < pieces; i += (int64_t)kRaClearGroups * kRaThreads) {
      const int64_t row = i / (p.heads * kPieces);
      const int at = (int)(i - row * (p.heads * kPieces)), h = at / kPieces, c = at % kPieces;
      uint16_t* dst = p.out + (row < first ? row : row - first + end) * p.out_stride_token + h * p.out_stride_head + 8 * c;
      *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
    }
    return;
  }

  // Item after item: a kv head after the other, so that with a multiple of eight heads the workgroups of an XCD (consecutive ones go to
  // different XCDs) read the same, and neighbouring tiles of a stream run side by side.  (Items handed to whoever asks first, by a counter
  // of each XCD that a launch ahead clears: 12 streams of 1 to 700 tokens over 300 to 9000 keys 176 us in turn, 199 so.)
  RaCursor<KIND == kRaListed ? kRaPaged : KIND, false> cursor;
  if constexpr (KIND != kRaListed) cursor.start(p);
  bool packed = false;  // each wave has an item of its own, of up to 32 rows
  RaList list{};
  uint32_t free_from = 0, round = 0;  // listed: the first workgroup that takes streams' items, how many times it did
  if constexpr (KIND == kRaListed) {
    list = *p.list;
    free_from = list.prefix_items < p.groups ? list.prefix_items : 0;
  }
  for (uint32_t id = blockIdx.x;; id += p.groups) {
  uint32_t index = id / (uint32_t)p.kv_heads, kv_head = id - index * (uint32_t)p.kv_heads;
  RaItem t;
  if constexpr (KIND == kRaListed) {
    uint32_t item = id;
    packed = false;
    if (item >= list.prefix_items) {
      // from the longest to the shortest, back and forth over the workgroups without a beginning
      if (blockIdx.x < free_from) return;
      const uint32_t free = p.groups - free_from, at = blockIdx.x - free_from;
      item = list.prefix_items + round * free + (round & 1 ? free - 1 - at : at);
      ++round;
      if (item >= list.single_items) {
        packed = true;
        item = list.single_items + 4 * (item - list.single_items);
        if (item >= list.items) return;
        item += threadIdx.x >> 6;
      }
    }
    __syncthreads();  // no wave is at the item before any more
    item = (uint32_t)__builtin_amdgcn_readfirstlane((int)item);
    if (packed && item >= list.items) continue;
    index = item / (uint32_t)p.kv_heads;
    kv_head = item - index * (uint32_t)p.kv_heads;
    const RaListedItem& of = p.listed[index];
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    t.rows = uniform(of.rows);
    t.q0 = uniform(of.q0);
    t.first = uniform(of.first);
    t.len = uniform(of.len);
    t.base = uniform(of.base);
    t.prefix_len = uniform(of.prefix_len);
    t.prefix_steps = steps_of(t.prefix_len);
    t.prefix_pages = p.prefix_table + (int64_t)uniform(of.prefix_row) * p.prefix_stride;
    t.pages = p.page_table + (int64_t)uniform(of.table_row) * p.table_stride;
    t.s_begin = uniform(of.s_begin);
    t.s_end = uniform(of.s_end);
    t.slot = uniform(of.slot);
    if (t.rows == 0) continue;
  } else {
  if (!cursor.find(p, index, t)) return;
  if (t.part >= t.n_parts) continue;  // a tile that sees fewer keys than the stream's last
  __syncthreads();                    // no wave is at the item before any more
  }
  // The thread's coordinates, formed anew for every item: what is derived from them would otherwise be formed ahead of the loop over the
  // items and take registers throughout.
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, lh = lane >> 5;
  const int s_begin = t.s_begin, s_end = t.s_end;
  const int tile_rows = min(kRaTileRows, t.rows - t.first);
  const uint16_t *k_head = p.k + kv_head * p.k_stride_head, *v_head = p.v + kv_head * p.v_stride_head;
  // As wider tiles, with three waves idle, up to 32 rows take longer: single tokens of 3 streams over up to 300 keys 9.7 us, so 7.8; of 32
  // streams over up to 16384 keys 118 us, so 108.
  const bool narrow = tile_rows <= 32;
  const int own = narrow ? 0 : wave * 32;  // the wave's first row in the tile

  // This lane's row.  Formed anew where it is needed at the end: over the loops it would take registers they do not have.
  struct Row {
    int token, head;
  };
  auto own_row = [&]() __attribute__((always_inline)) {
    int f = min(t.first + own + l32, t.rows - 1);
    asm volatile("" : "+v"(f));
    const int token = (uint32_t)f / p.group;
    return Row{token, (int)(kv_head * p.group.d) + f - token * (int)p.group.d};
  };
  const Row row = own_row();
  // what it sees: keys below `last`, from `from` on or below the sink
  const int pos = t.base + row.token;
  // (keys of a shared beginning have numbers below zero, and every row sees them)
  int last = p.causal ? min(pos + 1, t.len) : t.len;
  if constexpr (kPrefixed) last = max(last, 0);
  const int from = kPrefixed ? -(1 << 30) : p.window && pos >= (int)p.window ? pos - (int)p.window + 1 : 0;
  // the same for the wave's first and last row, which bound the others
  const int last0 = __builtin_amdgcn_readfirstlane(last), from1 = __builtin_amdgcn_readlane(from, 31);
  const bool idle = own >= tile_rows;  // a wave without rows only moves keys

  short8v qf[kSteps];
  float16v o[kDTiles];
#pragma unroll
  for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  bool finite = true;  // V where rows of the wave see different keys

  // ---- where the keys of 64 lanes lie
  uint8_t* const looked_up = smem + 4 * kStepBytes + wave * 512;
  const uint32_t looked_up_lds = lds_at(looked_up);
  auto key_base = [&](int s) __attribute__((always_inline)) {
    if constexpr (kPrefixed) return (s - t.prefix_steps) * kRaKeys;
    return (s < t.sink_steps ? s : t.from_step + s - t.sink_steps) * kRaKeys;
  };
  uint32_t next_row = 0;
  auto look_up = [&](int key, int slot) __attribute__((always_inline)) {
    uint32_t k = (uint32_t)min(key, t.len - 1);
    if constexpr (kPrefixed) {  // all 64 keys of a step lie on one side
      const bool shared = __builtin_amdgcn_readfirstlane(key) < 0;
      k = (uint32_t)min(shared ? key + t.prefix_steps * kRaKeys : key, (shared ? t.prefix_len : t.len) - 1);
      const uint32_t page = k / p.page;
      next_row = k - page * p.page.d;
      load4_to_lds((shared ? t.prefix_pages : t.pages) + page, looked_up_lds + slot * 256);
    }
    if constexpr (KIND == kRaPaged) {
      const uint32_t page = k / p.page;
      next_row = k - page * p.page.d;
      load4_to_lds(t.pages + page, looked_up_lds + slot * 256);
    }
    if constexpr (KIND == kRaMaskedRows) load4_to_lds(reinterpret_cast<const void*>((uintptr_t)(p.key_mask + t.key0 + k) & ~(uintptr_t)3), looked_up_lds + slot * 256);
  };
  uint32_t at_page = 0, at_row = 0;  // paged: page and row in it of this lane's key
  int first_key = 0;                 // the key of lane 0
  uint64_t there = 0;                // which of the 64 keys exist
  // The keys of the lanes: base + lane, or twice base + lane % 32.
  auto take_places = [&](int base, int at, int slot) __attribute__((always_inline)) {
    const int key = base + at;
    bool ok = key < t.len;
    if constexpr (kPrefixed) ok = base < 0 ? key + t.prefix_steps * kRaKeys < t.prefix_len : ok;
    first_key = base;
    if constexpr (kPages) {
      at_page = *reinterpret_cast<const uint32_t*>(looked_up + slot * 256 + lane * 4);
      at_row = next_row;  // of the key that was looked up last, which is this one where it exists
      ok = ok && at_page < p.n_pages;
    }
    if constexpr (KIND == kRaMaskedRows) {
      const uint32_t shift = 8 * ((uint32_t)(uintptr_t)(p.key_mask + t.key0 + min(key, t.len - 1)) & 3);
      ok = ok && ((*reinterpret_cast<const uint32_t*>(looked_up + slot * 256 + lane * 4) >> shift) & 0xFF) != 0;
    }
    there = __builtin_amdgcn_ballot_w64(ok);
  };

  // ---- loads: 16 rows, the keys of lanes r0 .. r0 + 15, to 16 rows of LDS
  // The lane's piece of row lane / kPieces of a load, and how its position turns from load to load.
  const uint32_t k_part = (uint32_t)k_piece<D>(lane / kPieces, lane % kPieces) * 16, v_part = (uint32_t)v_piece<D>(lane / kPieces, lane % kPieces) * 16;
  const uint32_t k_row = (uint32_t)(lane / kPieces) * p.k_stride_row * 2, v_row = (uint32_t)(lane / kPieces) * p.v_stride_row * 2;
  auto turn = [](bool values, int i) { return (values ? v_piece<D>(i * kRowsPerLoad, 0) : k_piece<D>(i * kRowsPerLoad, 0)) * 16; };
  typedef __attribute__((address_space(3))) u32x4* lds_uint4;
  // 16 rows from a multiple of 16 on lie one behind the other, and take one address for a wave in place of one for a lane: 532 x 40 / 8 heads
  // over 9000 keys in pages of 32 rows 118 us, of 24 rows 143.
  const bool whole_pages = kPages && p.page.d % 16 == 0;
  // counted: as many loads whatever keys there are, for waits that leave some under way.
  auto load_rows = [&](bool values, int r0, uint32_t lds, bool counted) __attribute__((always_inline)) {
    const uint16_t* base = values ? v_head : k_head;
    const uint32_t per_page = values ? p.v_stride_page : p.k_stride_page, per_row = values ? p.v_stride_row : p.k_stride_row;
    const uint32_t part = values ? v_part : k_part, in_row = values ? v_row : k_row;
    const uint32_t exist = (uint32_t)(there >> r0) & 0xFFFFu;
    // 16 rows one behind the other that may be read, whether they hold keys or not.
    bool in_line;
    uint64_t at;
    if constexpr (kPages) {
      in_line = whole_pages && (exist & 1);
      at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)at_page, r0) * per_page + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)at_row, r0) * per_row;
    } else {
      in_line = first_key + r0 < t.len && (int64_t)t.key0 + first_key + r0 + 15 < p.n_keys;
      at = (uint64_t)(uint32_t)(t.key0 + first_key + r0) * per_row;
    }
    if (in_line && (!values || exist == 0xFFFFu)) {  // K of keys that do not exist is read and not looked at
#pragma unroll
      for (int i = 0; i < kGroupLoads; ++i)
        load16_to_lds((part ^ (uint32_t)turn(values, i)) + in_row, uniform_pointer(base + at + (uint64_t)i * kRowsPerLoad * per_row), lds + i * 1024);
      return;
    }
    // What follows is rare enough to form the lane's places anew: kept over the loops they would take registers these do not have.
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int row0 = ln / kPieces, piece = ln % kPieces;
    if (in_line && !counted) {  // of V, zeros take the place of rows that hold no key
#pragma unroll
      for (int i = 0; i < kGroupLoads; ++i) {
        const int row = i * kRowsPerLoad + row0;
        if ((exist >> row) & 1) {  // lanes that take no part write nothing
          const uint32_t off = (uint32_t)row0 * per_row * 2 + (uint32_t)(values ? v_piece<D>(row, piece) : k_piece<D>(row, piece)) * 16;
          load16_to_lds(off, uniform_pointer(base + at + (uint64_t)i * kRowsPerLoad * per_row), lds + i * 1024);
        } else {
          *(lds_uint4)(uintptr_t)(lds + i * 1024 + ln * 16) = u32x4{0, 0, 0, 0};
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kGroupLoads; ++i) {
        const int in_group = i * kRowsPerLoad + row0, row = r0 + in_group;
        if constexpr (kPages) {
          at = (uint64_t)(uint32_t)__shfl((int)at_page, row) * per_page + (uint64_t)(uint32_t)__shfl((int)at_row, row) * per_row;
        } else {
          at = (uint64_t)(uint32_t)(t.key0 + first_key + row) * per_row;
        }
        const uint8_t* src = reinterpret_cast<const uint8_t*>(base + at) + (values ? v_piece<D>(in_group, piece) : k_piece<D>(in_group, piece)) * 16;
        load16_to_lds((there >> row) & 1 ? src : reinterpret_cast<const uint8_t*>(kRaZeros), lds + i * 1024);
      }
    }
  };

  // ---- scores and probabilities of NT groups of 32 keys from `base` on
  // S^T: register r of sc[kt] is key 32 kt + 8 (r / 4) + 4 lh + r % 4
  typedef const __attribute__((address_space(3))) short8v* lds_short8;
  typedef __attribute__((address_space(3))) short4v* lds_short4;
  typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
  typedef const __attribute__((address_space(3))) uint2v* lds_uint2;
  const uint32_t lds0 = lds_at(smem);
  // where the lane's fragments begin in LDS rows; a fragment's number turns bits of the piece's position
  const uint32_t k_lane = (uint32_t)(l32 * kRowBytes + k_piece<D>(l32, lh) * 16);
  auto read_k = [&](uint32_t k_rows, int kt, int ks) __attribute__((always_inline)) {
    return *(lds_short8)(uintptr_t)(((k_rows + k_lane) ^ (uint32_t)(32 * ks)) + 32 * kt * kRowBytes);
  };
  auto scores = [&](auto& sc, uint32_t k_rows) __attribute__((always_inline)) {
    constexpr int NT = std::extent<std::remove_reference_t<decltype(sc)>>::value;
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[kt][r] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        sc[kt] = T::mfma(read_k(k_rows, kt, ks), qf[ks], sc[kt]);
      }
    }
  };
  // Whether there are keys from `base` to `end` that a row of the wave does not see.
  auto uneven = [&](int base, int end) __attribute__((always_inline)) {
    if constexpr (kPrefixed) return min(end, t.len) > last0;
    return KIND == kRaPaged && (min(end, t.len) > last0 || (base < from1 && end > (int)p.sink));
  };
  auto seen_from = [&](int base) __attribute__((always_inline)) {  // of 64 keys from `base` on, those that the lane's row may see
    return low_bits(last - base) & (~low_bits(from - base) | low_bits((int)p.sink - base));
  };
  auto mask = [&](auto& sc, int base, uint64_t exist) __attribute__((always_inline)) {  // whether it hides any
    constexpr int NT = std::extent<std::remove_reference_t<decltype(sc)>>::value;
    constexpr uint64_t kAll = NT == 2 ? ~0ull : 0xFFFFFFFFull;
    const int end = base + 32 * NT;
    if ((exist & kAll) == kAll && !uneven(base, end)) return false;
    const uint64_t seen = exist & seen_from(base);  // one bit a key
    const uint32_t bits[2] = {(uint32_t)seen >> (4 * lh), (uint32_t)(seen >> 32) >> (4 * lh)};
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)bits[kt], 8 * (r / 4) + r % 4, 1);
        sc[kt][r] = __uint_as_float((keep & __float_as_uint(sc[kt][r])) | (~keep & 0xFF800000u));
      }
    return true;
  };
  float neg = 0.0f;
  auto largest = [&](auto& sc) __attribute__((always_inline)) {
    constexpr int NT = std::extent<std::remove_reference_t<decltype(sc)>>::value;
    float mx = sc[0][0];
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[kt][r]);
    return mx;
  };
  auto follow = [&](float mx) __attribute__((always_inline)) {  // the reference point for scores of which this lane's largest is mx
    mx = exchange_max(mx);
    const bool raise = (mx - m) * p.scale_log2 > kRaStep;
    if (__builtin_amdgcn_ballot_w64(raise) != 0) {
      float alpha;
      // a row that has seen nothing yet stays at -inf; 0 stands for it in the exponents, where -inf - -inf would be NaN
      if constexpr (T::kWeightShift == 0.0f) {
        alpha = raise ? __builtin_amdgcn_exp2f((m - mx) * p.scale_log2) : 1.0f;
        m = raise ? mx : m;
        neg = m == -INFINITY ? 0.0f : -m * p.scale_log2;
      } else {
        const float to = fmaf(-mx, p.scale_log2, weight_shift<T>(mx * p.scale_log2));
        alpha = raise && m != -INFINITY ? __builtin_amdgcn_exp2f(to - neg) : 1.0f;  // nothing seen: sums of zero stay what they are
        m = raise ? mx : m;
        neg = raise ? to : neg;
      }
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
  };
  // What the row's sums and outputs refer to, -inf for a row that has seen nothing.
  auto reference = [&]() __attribute__((always_inline)) { return T::kWeightShift == 0.0f || m == -INFINITY ? m : -neg; };
  // V^T of 16 keys and 32 columns: a lane needs column 32 dt + l32 of the keys 8 j + 4 lh + 0 .. 3 (j = 0, 1: the order of the scores'
  // registers).  A read serves 16 lanes: lane i points at row i / 4, columns 4 (i % 4) .. + 3, and each receives a column of the four rows.
  const uint32_t v_lane = (uint32_t)((4 * lh + ((lane & 15) >> 2)) * kRowBytes +
                                     v_piece<D>(4 * lh + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8);
  auto read_v = [&](uint32_t v_rows, int step, int dt, short4v (&dst)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      dst[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)(uintptr_t)(((v_rows + v_lane) ^ (uint32_t)(64 * dt)) + (16 * step + 8 * j) * kRowBytes));
  };
  auto weigh = [&](auto& sc, uint32_t v_rows) __attribute__((always_inline)) {
    constexpr int NT = std::extent<std::remove_reference_t<decltype(sc)>>::value;
#pragma unroll
    for (int step = 0; step < 2 * NT; ++step) {
      __builtin_amdgcn_sched_barrier(0);  // no reads of later steps ahead of this one: they would take the registers
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[step >> 1][8 * (step & 1) + 2 * u], p.scale_log2, neg));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[step >> 1][8 * (step & 1) + 2 * u + 1], p.scale_log2, neg));
        w[u] = T::pack2(p0, p1);  // at most 2^(kRaStep + kWeightShift): no overflow, and half a step's error each, as small as the result's own
        l = T::add2(w[u], l);     // the sum, in fp32, is of what the product weighs with
      }
      const short8v pb = __builtin_bit_cast(short8v, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) {
        short4v part[2];
        read_v(v_rows, step, dt, part);
        o[dt] = T::mfma(__builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7), pb, o[dt]);
      }
    }
  };
  // A key that some rows of the wave see and others do not: its weight of zero keeps it out of the others' sums, unless its V is not finite.
  // So where rows differ, V is looked through, and if it is not finite the item is done once more, rows of V that are not finite then being
  // added to the rows that see them alone.  (In a loop of its own: in the others it would take registers that they do not have.)
  auto all_finite = [&](uint32_t v_rows, int n_rows) __attribute__((always_inline)) {
    typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
    ushort2v top = {0, 0};
    for (int i = 0; i < n_rows * kRowBytes / 1024; ++i) {
      const u32x4 w = *(lds_uint4)(uintptr_t)(v_rows + i * 1024 + lane * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2v, w[j] & 0x7FFF7FFFu));
    }
    return __builtin_amdgcn_ballot_w64(top[0] >= T::kInfinity || top[1] >= T::kInfinity) == 0;
  };
  auto weigh_apart = [&](auto& sc, uint32_t v_rows, int base) __attribute__((always_inline)) {
    constexpr int NT = std::extent<std::remove_reference_t<decltype(sc)>>::value;
#pragma unroll
    for (int step = 0; step < 2 * NT; ++step) {
      __builtin_amdgcn_sched_barrier(0);
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[step >> 1][8 * (step & 1) + 2 * u], p.scale_log2, neg));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[step >> 1][8 * (step & 1) + 2 * u + 1], p.scale_log2, neg));
        w[u] = T::pack2(p0, p1);
        l = T::add2(w[u], l);
      }
      const short8v pb = __builtin_bit_cast(short8v, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) {
        short4v part[2];
        read_v(v_rows, step, dt, part);
        short8v a = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = (uint32_t)(a[j] & 0x7FFF) >= T::kInfinity ? (short)0 : a[j];
        o[dt] = T::mfma(a, pb, o[dt]);
      }
    }
    int ln = lane;
    asm volatile("" : "+v"(ln));  // formed here, not kept over the loops
    const uint64_t seen = seen_from(base);
#pragma unroll 1
    for (int j = 0; j < 32 * NT; ++j) {
      const bool sees = seen >> j & 1;
      const uint32_t row = v_rows + j * kRowBytes + (ln >> 5) * 8;
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {  // columns 32 dt + 8 g + 4 lh + 0 .. 3
          const uint2v v = *(lds_uint2)(uintptr_t)(row + v_piece<D>(j, 4 * dt + g) * 16);
          float x[4];
          T::unpack2(v[0], x[0], x[1]);
          T::unpack2(v[1], x[2], x[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[dt][4 * g + i] += sees && !(fabsf(x[i]) < INFINITY) ? x[i] : 0.0f;
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto once_more = [&]() __attribute__((always_inline)) {
    m = -INFINITY;
    l = neg = 0.0f;
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
  };
  // One step of a tile of more than 32 rows and the scores of the next: every slot one MFMA (S^T of the next step, then O^T of this one) with
  // what runs beside it, held in place by scheduling barriers: the LDS reads of MFMAs some slots later, and the probabilities, a pair
  // of keys' multiply-adds, exponentials and packing in three slots in a row.
  auto step_and_next = [&](float16v (&sc)[2], float16v (&nx)[2], uint32_t next_k, uint32_t v_rows) __attribute__((always_inline)) {
    constexpr int kS = 2 * kSteps, kSlots = kS + 4 * kDTiles, kAhead = D == 64 ? 2 : 4, kRing = kAhead + 1, kVAhead = D == 64 ? 2 : 3, kVRing = kVAhead + 1;
    short8v fk[kRing];
    short4v fv[kVRing][2];
    uint32_t pw[16];
    float x[2][2], e[2][2], mx = -INFINITY;
    auto fetch_k = [&](auto tag) __attribute__((always_inline)) {
      constexpr int i = decltype(tag)::value;
      fk[i % kRing] = read_k(next_k, i % 2, i / 2);
    };
    each_index(fetch_k, std::make_integer_sequence<int, kAhead>{});
    __builtin_amdgcn_sched_barrier(0);
    auto one_slot = [&](auto slot_tag) __attribute__((always_inline)) {
      constexpr int slot = decltype(slot_tag)::value;
      if constexpr (slot + kAhead < kS) fetch_k(std::integral_constant<int, slot + kAhead>{});
      if constexpr (slot + kVAhead >= kS && slot + kVAhead < kSlots) {
        constexpr int u = slot + kVAhead - kS;
        read_v(v_rows, u / kDTiles, u % kDTiles, fv[u % kVRing]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (slot < kS) {
        constexpr int kt = slot % 2, ks = slot / 2;
        const float16v zero = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        nx[kt] = T::mfma(fk[slot % kRing], qf[ks], ks == 0 ? zero : nx[kt]);
      } else {
        constexpr int u = slot - kS, step = u / kDTiles, dt = u % kDTiles;
        const short4v(&v)[2] = fv[u % kVRing];
        const short8v pb = __builtin_bit_cast(short8v, make_uint4(pw[4 * step], pw[4 * step + 1], pw[4 * step + 2], pw[4 * step + 3]));
        o[dt] = T::mfma(__builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7), pb, o[dt]);
      }
      // pair i of the 16 pairs of keys begins in slot i * kSlots * 3 / 64
      auto pairs = [&](auto pair_tag) __attribute__((always_inline)) {
        constexpr int pair = decltype(pair_tag)::value, begin = pair * kSlots * 3 / 64;
        if constexpr (slot == begin + 2) {
          pw[pair] = T::pack2(e[pair & 1][0], e[pair & 1][1]);  // no overflow, see weigh
          asm volatile("" : "+v"(pw[pair]));                    // here, and not sunk to the MFMA that reads it
          l = T::add2(pw[pair], l);
        }
        if constexpr (slot == begin + 1) {
          e[pair & 1][0] = __builtin_amdgcn_exp2f(x[pair & 1][0]);
          e[pair & 1][1] = __builtin_amdgcn_exp2f(x[pair & 1][1]);
        }
        if constexpr (slot == begin) {
          constexpr int kt = pair >> 3, r = 2 * (pair & 7);
          x[pair & 1][0] = fmaf(sc[kt][r], p.scale_log2, neg);
          x[pair & 1][1] = fmaf(sc[kt][r + 1], p.scale_log2, neg);
        }
      };
      each_index(pairs, std::make_integer_sequence<int, 16>{});
      // the next scores' largest, in the second half of the slots, two slots behind the last product of a group of keys
      if constexpr (slot >= kSlots / 2 + 2) {
        constexpr int first = (slot - kSlots / 2 - 2) * 32 / (kSlots / 2 - 2), end = (slot - kSlots / 2 - 1) * 32 / (kSlots / 2 - 2);
#pragma unroll
        for (int i = first; i < end; ++i) mx = fmaxf(mx, nx[i >> 4][i & 15]);
        asm volatile("" : "+v"(mx));
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    each_index(one_slot, std::make_integer_sequence<int, kSlots>{});
    return mx;
  };

  const bool to_record = KIND == kRaListed ? t.slot >= 0 : t.n_parts > 1;
  auto write_record = [&](int row_in_tile, int column, const float (&v)[4], float mm, float ll) __attribute__((always_inline)) {
    // four columns of a row of this part's record
    if constexpr (KIND == kRaListed) {
      const int f = t.first + row_in_tile, token = (uint32_t)f / p.group, head = kv_head * p.group.d + (f - token * p.group.d);
      const uint32_t slot = (uint32_t)t.slot;
      *reinterpret_cast<float4*>(shared_record<D>(p, slot, t.q0 + token, head) + column) = make_float4(v[0], v[1], v[2], v[3]);
      if (column == 0) *shared_sums<D>(p, slot, t.q0 + token, head) = make_float2(mm, ll);
      return;
    }
    *reinterpret_cast<float4*>(record_of<D>(p, kv_head, t, t.part, row_in_tile) + column) = make_float4(v[0], v[1], v[2], v[3]);
    if (column == 0) *record_sums<D>(p, kv_head, t, t.part, row_in_tile) = make_float2(mm, ll);
  };

  if (!narrow) {
    // K of step s is in buffer s & 1 an iteration before V of step s is: scores are a step ahead.
    const uint32_t k_lds = lds0 + wave * 16 * kRowBytes, v_lds = k_lds + 2 * kStepBytes;
    auto load_k = [&](int s) __attribute__((always_inline)) {
      take_places(key_base(s), lane, s & 1);
      load_rows(false, wave * 16, k_lds + (s & 1) * kStepBytes, false);
      if (kLooksUp && s + 1 < s_end) look_up(key_base(s + 1) + lane, (s + 1) & 1);
    };
    auto load_v = [&](int s) __attribute__((always_inline)) { load_rows(true, wave * 16, v_lds + (s & 1) * kStepBytes, false); };
    const uint32_t k_rows = lds0, v_rows = lds0 + 2 * kStepBytes;
    uint64_t exist = 0;
    if (s_begin < s_end) {
      // The wave's queries, whole rows per load, by way of the buffers that the first step leaves alone: straight into the fragments a load
      // reaches 32 bytes of each of 32 rows.
      const uint32_t q_lds = (wave < 2 ? k_rows : v_rows) + ((s_begin & 1) ^ 1) * kStepBytes + (wave & 1) * 32 * kRowBytes;
      if (!idle) {
#pragma unroll
        for (int i = 0; i < 2 * kGroupLoads; ++i) {
          const int r = i * kRowsPerLoad + lane / kPieces, f = min(t.first + own + r, t.rows - 1);
          const int token = (uint32_t)f / p.group, head = (int)(kv_head * p.group.d) + f - token * (int)p.group.d;
          load16_to_lds(p.q + (t.q0 + token) * p.q_stride_token + head * p.q_stride_head + 8 * k_piece<D>(r, lane % kPieces), q_lds + i * 1024);
        }
      }
      if (kLooksUp) {
        look_up(key_base(s_begin) + lane, s_begin & 1);
        wait_loads<0>();
      }
      load_k(s_begin);
      exist = there;
      load_v(s_begin);
      wait_loads<0>();
      if (!idle) {
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) qf[ks] = read_k(q_lds, 0, ks);
      }
      __syncthreads();
      if (s_begin + 1 < s_end) load_k(s_begin + 1);
    }
    // An iteration's loads: K of step s + 1 and V of step s are in LDS, and every wave is done with K of step s and V of step s - 1.
    auto move_keys = [&](int s) __attribute__((always_inline)) {
      wait_loads<0>();
      __syncthreads();
      exist = there;  // of step s + 1
      load_v(s + 1);  // from the places of the last load_k
      if (s + 2 < s_end) load_k(s + 2);
    };
    // The item once more, step by step (see all_finite).
    auto apart = [&]() __attribute__((always_inline)) {
      once_more();
#pragma unroll 1
      for (int s = s_begin; s < s_end; ++s) {
        __syncthreads();
        if (kLooksUp) {
          look_up(key_base(s) + lane, 0);
          wait_loads<0>();
        }
        take_places(key_base(s), lane, 0);
        load_rows(false, wave * 16, k_lds, false);
        load_rows(true, wave * 16, v_lds, false);
        wait_loads<0>();
        __syncthreads();
        if (idle) continue;
        float16v sc[2];
        scores(sc, k_rows);
        mask(sc, key_base(s), there);
        follow(largest(sc));
        weigh_apart(sc, v_rows, key_base(s));
      }
      __syncthreads();
    };
    const bool may_differ = kPages && (p.causal || p.window);
    if (idle) {
      if (s_begin < s_end) {
        for (int s = s_begin; s + 1 < s_end; ++s) move_keys(s);
        wait_loads<0>();
        __syncthreads();
        if (may_differ && __syncthreads_or(0)) apart();
      }
      continue;
    }
    if (s_begin < s_end) {
      float16v sc[2][2];
      scores(sc[0], k_rows + (s_begin & 1) * kStepBytes);
      mask(sc[0], key_base(s_begin), exist);
      follow(largest(sc[0]));
      auto iteration = [&](int s, auto from_tag) __attribute__((always_inline)) {
        constexpr int from_buffer = decltype(from_tag)::value;
        move_keys(s);
        const uint32_t next_k = k_rows + ((s + 1) & 1) * kStepBytes, this_v = v_rows + (s & 1) * kStepBytes;
        if (uneven(key_base(s), key_base(s) + kRaKeys)) finite = finite && all_finite(this_v, kRaKeys);
        float mx = step_and_next(sc[from_buffer], sc[from_buffer ^ 1], next_k, this_v);
        if (mask(sc[from_buffer ^ 1], key_base(s + 1), exist)) mx = largest(sc[from_buffer ^ 1]);
        follow(mx);
      };
      int s = s_begin;
      for (; s + 2 < s_end; s += 2) {
        iteration(s, std::integral_constant<int, 0>{});
        iteration(s + 1, std::integral_constant<int, 1>{});
      }
      if (s + 1 < s_end) {
        iteration(s, std::integral_constant<int, 0>{});
        sc[0][0] = sc[1][0];
        sc[0][1] = sc[1][1];
        ++s;
      }
      wait_loads<0>();
      __syncthreads();
      const uint32_t this_v = v_rows + (s & 1) * kStepBytes;
      if (uneven(key_base(s), key_base(s) + kRaKeys)) finite = finite && all_finite(this_v, kRaKeys);
      weigh(sc[0], this_v);
      if (may_differ && __syncthreads_or(!finite)) apart();
    }
    l = exchange_sum(l);
    if (to_record) {
      if (own + l32 < tile_rows) {
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float v[4] = {o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
            write_record(own + l32, 32 * dt + 8 * g + 4 * lh, v, reference(), l);
          }
      }
      continue;
    }
    // Whole rows per store, through the buffers of K, which every wave left ahead of the last step's barrier: straight from the registers a
    // store reaches 16 bytes of each of 32 rows.
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint8_t* patch = smem + wave * 32 * kRowBytes;
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint2*>(patch + l32 * kRowBytes + k_piece<D>(l32, 4 * dt + g) * 16 + lh * 8) =
            make_uint2(T::pack2(o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv), T::pack2(o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int it = 0; it < 32 / kRowsPerLoad; ++it) {
      const int r = it * kRowsPerLoad + lane / kPieces, piece = lane % kPieces;
      const uint4 v = *reinterpret_cast<const uint4*>(patch + r * kRowBytes + k_piece<D>(r, piece) * 16);
      if (own + r < tile_rows) {
        const int f = t.first + own + r, token = (uint32_t)f / p.group, head = kv_head * p.group.d + (f - token * p.group.d);
        *reinterpret_cast<uint4*>(p.out + (t.q0 + token) * p.out_stride_token + head * p.out_stride_head + 8 * piece) = v;
      }
    }
    continue;
  }

  // ---- up to 32 rows: groups of 32 keys u = 2 s + half, every fourth one this wave's
  const uint32_t rows_lds = lds0 + wave * kStepBytes;  // 32 rows of K, 32 of V
  constexpr int kLoads = 2 * kGroupLoads;  // of K or of V
  auto group_base = [&](int u) __attribute__((always_inline)) { return key_base(u >> 1) + 32 * (u & 1); };
  auto load_group = [&](bool values) __attribute__((always_inline)) {
    load_rows(values, 0, rows_lds + (values ? 32 * kRowBytes : 0), true);
    load_rows(values, 16, rows_lds + (values ? 32 * kRowBytes : 0) + 16 * kRowBytes, true);
  };
  const int u_end = 2 * s_end, u_first = 2 * s_begin + (KIND == kRaListed && packed ? 0 : wave), u_step = KIND == kRaListed && packed ? 1 : 4;
  int u = u_first;
  {
    const uint16_t* src = p.q + (t.q0 + row.token) * p.q_stride_token + row.head * p.q_stride_head + 8 * lh;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) qf[ks] = *reinterpret_cast<const short8v*>(src + 16 * ks);
  }
  if (u < u_end) {
    if (kLooksUp) {
      look_up(group_base(u) + l32, 0);
      wait_loads<0>();
    }
    take_places(group_base(u), l32, 0);
    load_group(false);
    if (kLooksUp) look_up(group_base(min(u + u_step, u_end - 1)) + l32, 1);
    load_group(true);
  }
  // Ahead of the loop and where the compiler sees it: it would otherwise count the loads of the queries as under way for good, and wait
  // for the keys' loads in their place ahead of every product.  0x0F70 = vmcnt(0), other counters untouched.
  __builtin_amdgcn_s_waitcnt(0x0F70);
  if (u < u_end) {
    for (int slot = 1; u < u_end; u += u_step, slot ^= 1) {
      const uint64_t exist = there;
      const bool more = u + u_step < u_end;
      wait_loads<kLoads>();  // K, and the places of the next group; V may be on its way
      float16v sc[1];
      scores(sc, rows_lds);
      if (more) {
        take_places(group_base(u + u_step), l32, slot);
        wait_lds_reads();
        load_group(false);
        if (kLooksUp) look_up(group_base(min(u + 2 * u_step, u_end - 1)) + l32, slot ^ 1);
      }
      mask(sc, group_base(u), exist);
      follow(largest(sc));
      if (more) wait_loads<kLoads + (kLooksUp ? 1 : 0)>();
      else wait_loads<0>();
      const uint32_t this_v = rows_lds + 32 * kRowBytes;
      if (uneven(group_base(u), group_base(u) + 32)) finite = finite && all_finite(this_v, 32);
      weigh(sc, this_v);
      if (more) {
        wait_lds_reads();
        load_group(true);
      }
    }
  }
  if (kPages && !finite) {  // once more, group by group (see all_finite)
    once_more();
#pragma unroll 1
    for (u = u_first; u < u_end; u += u_step) {
      if (kLooksUp) {
        look_up(group_base(u) + l32, 0);
        wait_loads<0>();
      }
      take_places(group_base(u), l32, 0);
      wait_lds_reads();
      load_group(false);
      load_group(true);
      wait_loads<0>();
      float16v sc[1];
      scores(sc, rows_lds);
      mask(sc, group_base(u), there);
      follow(largest(sc));
      weigh_apart(sc, rows_lds + 32 * kRowBytes, group_base(u));
    }
  }
  l = exchange_sum(l);
  if (KIND == kRaListed && packed) {
    const Row to = own_row();
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (l32 < tile_rows) {
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float v[4] = {o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
          const int column = 32 * dt + 8 * g + 4 * lh;
          if (to_record) write_record(l32, column, v, reference(), l);
          else
            *reinterpret_cast<uint2*>(p.out + (t.q0 + to.token) * p.out_stride_token + to.head * p.out_stride_head + column) =
                make_uint2(T::pack2(v[0] * inv, v[1] * inv), T::pack2(v[2] * inv, v[3] * inv));
        }
    }
    continue;
  }
  // The four waves' results, joined: each wave takes a quarter of the columns.
  float2* const ml = reinterpret_cast<float2*>(smem + 4 * kStepBytes + 4 * 512);
  if (lh == 0) ml[wave * 32 + l32] = make_float2(reference(), l);
  {
    float4* mine = reinterpret_cast<float4*>(smem + wave * kStepBytes);
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) mine[(dt * 4 + g) * 64 + lane] = make_float4(o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]);
  }
  __syncthreads();
  const Row to = own_row();
  float weight[4], all_l = 0.0f, all_m = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) all_m = fmaxf(all_m, ml[w * 32 + l32].x);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 e = ml[w * 32 + l32];
    weight[w] = e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((e.x - all_m) * reference_unit<T>(p.scale_log2));
    // a row without a reference point of which the sum is NaN has met NaN only
    all_l += e.x == -INFINITY ? e.y : e.y * weight[w];
  }
  const float inv = all_l == 0.0f ? 0.0f : 1.0f / all_l;
#pragma unroll
  for (int i = 0; i < kDTiles; ++i) {
    const int piece = wave * kDTiles + i, dt = piece >> 2, g = piece & 3;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float4 e = reinterpret_cast<const float4*>(smem + w * kStepBytes)[piece * 64 + lane];
      v[0] = fmaf(e.x, weight[w], v[0]);
      v[1] = fmaf(e.y, weight[w], v[1]);
      v[2] = fmaf(e.z, weight[w], v[2]);
      v[3] = fmaf(e.w, weight[w], v[3]);
    }
    const int column = 32 * dt + 8 * g + 4 * lh;
    if (l32 < tile_rows && to_record) write_record(l32, column, v, all_m, all_l);
    if (l32 < tile_rows && !to_record)
      *reinterpret_cast<uint2*>(p.out + (t.q0 + to.token) * p.out_stride_token + to.head * p.out_stride_head + column) =
          make_uint2(T::pack2(v[0] * inv, v[1] * inv), T::pack2(v[2] * inv, v[3] * inv));
  }
  }
}

// Joins the parts of the tiles that were cut, item by item: D / 4 lanes a row.
template <typename T, int D, int KIND>
__global__ __launch_bounds__(kRaThreads) void ragged_join_kernel(RaParams p) {
  constexpr int kRows = kRaThreads * 4 / D;
  const int column = threadIdx.x % (D / 4) * 4;
  RaCursor<KIND, true> cursor;
  cursor.start(p);
  for (uint32_t id = blockIdx.x;; id += gridDim.x) {
    const uint32_t index = id / (uint32_t)p.kv_heads, kv_head = id - index * (uint32_t)p.kv_heads;
    RaItem t;
    if (!cursor.find(p, index, t)) return;
    if (t.n_parts == 1) continue;
    const int rows = min(kRaTileRows, t.rows - t.first);
    for (int row = blockIdx.y * kRows + threadIdx.x / (D / 4); row < rows; row += gridDim.y * kRows) {
      float m = -INFINITY, l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int part = 0; part < t.n_parts; ++part) {
        const float2 e = *record_sums<D>(p, kv_head, t, part, row);
        const float4 y = *reinterpret_cast<const float4*>(record_of<D>(p, kv_head, t, part, row) + column);
        const float top = fmaxf(m, e.x);
        const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * reference_unit<T>(p.scale_log2));
        const float b = e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((e.x - top) * reference_unit<T>(p.scale_log2));
        // a sum beside a reference of -inf is zero, or NaN where NaN was all that was met
        l = (m == -INFINITY ? l : l * a) + (e.x == -INFINITY ? e.y : e.y * b);
        v[0] = fmaf(y.x, b, v[0] * a);
        v[1] = fmaf(y.y, b, v[1] * a);
        v[2] = fmaf(y.z, b, v[2] * a);
        v[3] = fmaf(y.w, b, v[3] * a);
        m = top;
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int f = t.first + row, token = (uint32_t)f / p.group, head = kv_head * p.group.d + (f - token * p.group.d);
      uint16_t* dst = p.out + (t.q0 + token) * p.out_stride_token + head * p.out_stride_head + column;
      *reinterpret_cast<uint2*>(dst) = make_uint2(T::pack2(v[0] * inv, v[1] * inv), T::pack2(v[2] * inv, v[3] * inv));
    }
  }
}

// ---- beginnings that groups attend together
//
// The rows of a joined group attend the beginning as tiles of their own, each stream's rows its own keys, and a last launch joins the two, row by
// row.  What all this takes is known to the device alone, so a launch of one workgroup adds it up and lists the items: first the beginnings', in
// parts, then the streams' own.  On a unit tiles of few rows, which wait for memory, then run beside wide ones.  A wave by itself takes two to
// three times as long for a narrow tile as four do together, waiting for the page table, then for K, for little else: four tiles run side by
// side, if one does not take longer than the launch does anyway.
//
// What bounds it, next to the floor of reading every key once or of all products at the library's rate: the three launches one behind the other, and
// items whose beginning is a chain of waits (places, keys, scores), so that the shortest takes 5 us and a workgroup has three to five of them.  Calls
// one behind the other; in brackets list, items and joining by a kernel trace, under which all three take up to an eighth longer: 64 single tokens x 32 / 8
// heads of 128 columns over 16384 shared and 30 to 1000 own keys 60 us, 52 with keys from the last-level cache (8, 43, 8), where 140 MB copied take 28.5;
// each stream over all of its keys takes 354.  100 x 4 tokens x 12 heads of 64 over 3001 and 8 to 300 keys 39 (7, 27, 7), copied 8.6; 104.  41 streams
// of 1 to 200 tokens x 20 / 4 of 128 in four groups, over 300 to 5000 and 10 to 900, 76 (9, 61, 15), the library's products 16.5; 85.  4 x 2640
// tokens x 24 over 10560 and 2640 are not joined, since their tiles are full as they are: 1740 to 1790, 0.96 to 0.98 PFLOP/s.
//
// us of 64 single tokens x 32 / 8 heads over 16384 shared and 30 to 1000 own keys: items found by every workgroup in turn, beginnings first, in 32
// parts 62, in 14 parts 63; so on workgroups of their own 50.
constexpr int kRaPlanThreads = 256;   // a wave to a SIMD: 64 streams 8.6 us, with four waves, most of them idle, 10.9
constexpr int kRaJoinedGroups = 256;  // in a launch at most: a thread each
constexpr int kRaSizes = 64;
constexpr int kRaLeastPrefixPart = 2, kRaLeastOwnPart = 5;  // steps

// us, by columns: of a wide tile's beginning, of its steps with up to one, two and three of them on a unit, of a narrow tile by four waves and by one,
// of joining a part of a wide tile (of the whole device).
struct RaCosts {
  float wide, wide_step[3], narrow, narrow_step, alone, alone_step, join;
};
__device__ __forceinline__ constexpr RaCosts costs_of(int columns) {
  return columns == 128 ? RaCosts{7.0f, {1.8f, 2.3f, 2.3f}, 5.5f, 1.3f, 3.4f, 3.3f, 0.0135f} : RaCosts{4.0f, {1.4f, 1.7f, 2.0f}, 4.2f, 0.95f, 4.1f, 2.65f, 0.007f};
}

struct RaSharedStream {
  int q0, rows, len, base, shares, prefix_len, joined;
};
__device__ __forceinline__ RaSharedStream shared_stream(const RaParams& p, int b) {  // but for its group
  RaSharedStream s;
  const int limit = (int)p.n_queries;
  const int start = p.q_starts[b], next = p.q_starts[b + 1];
  const int64_t given = max((int64_t)p.kv_lens[b], (int64_t)0);
  s.q0 = min(max(start, 0), limit);
  s.rows = max(min(max(next, 0), limit) - s.q0, 0) * (int)p.group.d;
  s.len = (int)min(given, p.table_keys);
  s.base = (int)(given - ((int64_t)next - s.q0));
  s.shares = -1;
  s.prefix_len = s.joined = 0;
  return s;
}
// Steps of a tile whose last row is `last_row` of its stream's, over the stream's own keys.
__device__ __forceinline__ int own_steps_of(const RaParams& p, const RaSharedStream& s, int last_row) {
  const int end = p.causal ? min(s.base + (int)((uint32_t)last_row / p.group) + 1, s.len) : s.len;
  return end > 0 ? steps_of(end) : 0;
}

__device__ __forceinline__ float sum_upto(float v) {  // over this lane and those before it
#define LL_DPP_ADD(ctrl, row_mask) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, row_mask, 0xF, true))
  LL_DPP_ADD(0x111, 0xF);
  LL_DPP_ADD(0x112, 0xF);
  LL_DPP_ADD(0x114, 0xF);
  LL_DPP_ADD(0x118, 0xF);
  LL_DPP_ADD(0x142, 0xA);
  LL_DPP_ADD(0x143, 0xC);
#undef LL_DPP_ADD
  return v;
}
template <typename V>
__device__ __forceinline__ V of_lane(V v, int lane) {
  return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// Sums over the threads of the planning workgroup, N at once: v becomes those before this thread, `all` those of all.
template <typename V, int N>
__device__ __forceinline__ void plan_sums(V (&v)[N], V (&all)[N], V (&of_waves)[N][kRaPlanThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  V upto[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    upto[i] = sum_upto(v[i]);
    if (lane == 63) of_waves[i][wave] = upto[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const V waves = sum_upto(lane < kRaPlanThreads / 64 ? of_waves[i][lane] : (V)0);
    all[i] = of_lane(waves, kRaPlanThreads / 64 - 1);
    v[i] = upto[i] - v[i] + (wave ? of_lane(waves, max(wave - 1, 0)) : (V)0);
  }
  __syncthreads();
}

template <int D>
__global__ __launch_bounds__(kRaPlanThreads) void shared_plan_kernel(RaParams p, uint32_t units) {
  constexpr RaCosts cost = costs_of(D);
  __shared__ int starts[kRaJoinedGroups + 1], lens[kRaJoinedGroups], group_q0[kRaJoinedGroups], group_rows[kRaJoinedGroups];  // lens below zero: joined
  __shared__ uint32_t upto[kRaJoinedGroups], sizes[2 * kRaSizes];  // items up to a group; of so long, for a workgroup and for a wave
  __shared__ float floats[5][kRaPlanThreads / 64];
  __shared__ uint32_t words[1][kRaPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  // threads of a stream, for its tiles, and streams at a time
  const int per_stream = p.streams <= 16 ? 16 : p.streams <= 32 ? 8 : p.streams <= 64 ? 4 : p.streams <= 128 ? 2 : 1, at_once = kRaPlanThreads / per_stream;
  const int tile0 = tid % per_stream, mine = tid / per_stream;
  const RaSharedStream early = shared_stream(p, min(mine, p.streams - 1));
  float take[5] = {};  // beginnings; wide tiles, narrow ones by four waves, by one; how many of these
  if (tid < p.n_groups) {
    const RaGroup r = group_of(p, tid);
    const int rows = r.n * (int)p.group.d;
    starts[tid] = p.group_starts ? p.group_starts[tid] : 0;
    if (tid == p.n_groups - 1) starts[tid + 1] = p.group_starts ? p.group_starts[tid + 1] : p.streams;
    lens[tid] = r.joined ? -r.len : r.len;
    group_q0[tid] = r.q0;
    group_rows[tid] = rows;
    if (r.joined) take[0] = (float)tiles_of(rows) * (float)steps_of(r.len) * (rows <= 32 ? cost.narrow_step : cost.wide_step[0]);
  }
  __syncthreads();
  const auto with_group = [&](RaSharedStream s, int b) __attribute__((always_inline)) {
    if (b >= p.streams) s.rows = 0;
    int g = 0, end = p.n_groups + 1;
    while (end - g > 1) {
      const int at = (g + end) >> 1;
      if (starts[at] <= b) g = at;
      else end = at;
    }
    if (g == p.n_groups || starts[g] > b) return s;
    s.shares = g;
    s.joined = lens[g] < 0;
    s.prefix_len = max(lens[g], 0);
    return s;
  };
  const RaSharedStream first = with_group(early, mine);
  const auto stream = [&](int b0) __attribute__((always_inline)) {  // of this thread
    return b0 == 0 ? first : with_group(shared_stream(p, min(b0 + mine, p.streams - 1)), b0 + mine);
  };
  const auto steps_in = [](const RaSharedStream& s) { return steps_of(s.prefix_len) + steps_of(s.len); };
  // ---- what there is to do, in us of a workgroup
  for (int b0 = 0; b0 < p.streams; b0 += at_once) {
    const RaSharedStream s = stream(b0);
    const int steps = steps_in(s);
    if (tile0 != 0 || s.rows == 0 || (s.joined && steps == 0)) continue;
    if (s.rows <= 32) {
      take[2] += cost.narrow + cost.narrow_step * steps;
      take[3] += cost.alone + cost.alone_step * steps;
      take[4] += 1.0f;
    } else {
      take[1] += (float)tiles_of(s.rows) * (cost.wide + cost.wide_step[1] * steps);
    }
  }
  float all_take[5];
  plan_sums(take, all_take, floats);
  const float heads = (float)p.kv_heads, prefixes = all_take[0] * heads, wide = all_take[1] * heads, narrow = all_take[2] * heads, alone = all_take[3] * heads,
              tiles = all_take[4] * heads;
  // us with four waves to each / one: 128 single tokens of five groups x 32 / 8 heads (1024 tiles for 512 workgroups) over 20 to 2000 own keys 99.2 /
  // 87.8, 100 x 40 / 8 over 20 to 60 30.6 / 29.4, 32 x 24 over 20 to 600 50.5 / 49.1; 64 x 32 / 8 over 30 to 1000 (512 tiles) 51.6 / 57.4, 20 of 1 to
  // 64 tokens x 24 over 10 to 400 (some 300 narrow ones) 51.9 / 63.9.
  const bool pack = tiles >= 1.4f * p.groups && alone * p.groups <= 2.0f * tiles * (prefixes + wide + 0.25f * alone);
  // ---- the streams' items, of about half of what a workgroup has to do: how many there are of about as much, what they take
  const float estimate = (prefixes + wide + (pack ? 0.25f * alone : narrow)) / p.groups, per_us = 0.75f * kRaSizes / fmaxf(estimate, 1.0f);
  const auto part_within = [&](float start, float step) { return (uint32_t)max((int)fminf((0.5f * estimate - start) / step, 1e9f), kRaLeastOwnPart); };
  const uint32_t wide_own = part_within(cost.wide, cost.wide_step[1]), narrow_own = pack ? part_within(cost.alone, cost.alone_step) : part_within(cost.narrow, cost.narrow_step);
  // What an item takes, in 65536ths of a size: whole numbers, since it has to come out the same where it is counted and where it is listed.
  struct Size {
    uint32_t start, step;
  };
  const auto sizes_of = [&](float start, float step) {
    const auto whole = [&](float us) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(65536.0f * us * per_us)); };
    return Size{whole(start), whole(step)};
  };
  const Size wide_size = sizes_of(cost.wide, cost.wide_step[1]), narrow_size = pack ? sizes_of(cost.alone, cost.alone_step) : sizes_of(cost.narrow, cost.narrow_step);
  if (tid < 2 * kRaSizes) sizes[tid] = 0;
  __syncthreads();
  // f(class, size, steps of the tile, its parts, steps of each, us of each) for every tile of a stream that has something to do
  const auto each_tile = [&](const RaSharedStream& s, auto&& f) __attribute__((always_inline)) {
    for (int tile = tile0; tile < tiles_of(s.rows); tile += per_stream) {
      const int steps = steps_of(s.prefix_len) + own_steps_of(p, s, min(tile * kRaTileRows + kRaTileRows, s.rows) - 1);
      if (s.joined && steps == 0) continue;  // nothing to add; one that is not joined has its zeros to write
      const int parts = max(shared_parts((uint32_t)steps, s.rows <= 32 ? narrow_own : wide_own, p.own_parts), 1), part = parts > 1 ? (steps + parts - 1) / parts : steps;
      const bool by_wave = pack && s.rows <= 32;
      const Size z = s.rows <= 32 ? narrow_size : wide_size;
      const float us = s.rows > 32 ? cost.wide + cost.wide_step[1] * part : by_wave ? 0.25f * (cost.alone + cost.alone_step * part) : cost.narrow + cost.narrow_step * part;
      f(tile, by_wave ? 1 : 0, kRaSizes - 1 - (int)min((z.start + (uint64_t)z.step * (uint32_t)part) >> 16, (uint64_t)kRaSizes - 1), steps, parts, part, us);
    }
  };
  float takes_now[1] = {0.0f}, takes_all[1];
  for (int b0 = 0; b0 < p.streams; b0 += at_once) {
    const RaSharedStream s = stream(b0);
    each_tile(s, [&](int, int by_wave, int size, int, int parts, int, float us) {
      atomicAdd(&sizes[by_wave * kRaSizes + size], (uint32_t)parts);
      takes_now[0] += parts * us;
    });
  }
  plan_sums(takes_now, takes_all, *reinterpret_cast<float(*)[1][kRaPlanThreads / 64]>(&floats));
  const float streams_take = takes_all[0] * heads;
  // ---- steps of a part of a beginning: a lane to a number of them, about a workgroup's share.  Which one has all done first?
  const int steps_tried = max((int)fminf((prefixes + streams_take) / p.groups / cost.wide_step[0] * (0.3f + 0.05f * lane), 1e9f), kRaLeastPrefixPart);
  uint32_t prefix_part;
  {
    uint32_t items = 0;
    int wide_part = 0, narrow_part = 0;
    float rows = 0.0f;
    for (int g = 0; g < p.n_groups; ++g) {
      if (lens[g] >= 0 || group_rows[g] == 0) continue;
      const int steps = steps_of(-lens[g]), n = shared_parts((uint32_t)steps, (uint32_t)steps_tried, p.prefix_parts), part = (steps + n - 1) / n;
      items += (uint32_t)(tiles_of(group_rows[g]) * n);
      rows += (float)group_rows[g] * n;
      if (group_rows[g] <= 32) narrow_part = max(narrow_part, part);
      else wide_part = max(wide_part, part);
    }
    items *= (uint32_t)p.kv_heads;
    const float step = cost.wide_step[items <= units ? 0 : items <= 2 * units ? 1 : 2];
    const float one = fmaxf(wide_part ? cost.wide + step * wide_part : 0.0f, narrow_part ? cost.narrow + cost.narrow_step * narrow_part : 0.0f);
    const float takes = rows * heads * (cost.join / kRaTileRows) +
                        (items < p.groups ? fmaxf(one, streams_take / (p.groups - items)) : one * ((items + p.groups - 1) / p.groups) + streams_take / p.groups);
    float least = takes;
    for (int i = 1; i < 64; i <<= 1) least = fminf(least, __shfl_xor(least, i));
    const int best = __builtin_ctzll(__builtin_amdgcn_ballot_w64(takes <= least) | (1ull << 63));
    prefix_part = (uint32_t)__builtin_amdgcn_readlane(steps_tried, best);
  }
  for (int b0 = 0; b0 < p.streams; b0 += at_once) {
    const RaSharedStream s = stream(b0);
    if (tile0 == 0 && b0 + mine < p.streams)
      p.joined[b0 + mine] = RaJoined{s.joined ? shared_parts((uint32_t)steps_of(-lens[s.shares]), prefix_part, p.prefix_parts) : 0, steps_of(s.prefix_len), s.joined};
  }
  uint32_t of_groups[1] = {}, all_of_groups[1];
  if (tid < p.n_groups && lens[tid] < 0)
    of_groups[0] = (uint32_t)(tiles_of(group_rows[tid]) * shared_parts((uint32_t)steps_of(-lens[tid]), prefix_part, p.prefix_parts));
  const uint32_t of_group = of_groups[0];
  plan_sums(of_groups, all_of_groups, words);
  // ---- the items of the beginnings
  const uint32_t prefix_items = min(all_of_groups[0], p.most_listed);
  if (tid < p.n_groups) upto[tid] = of_groups[0] + of_group;
  __syncthreads();
  for (uint32_t i = tid; i < prefix_items; i += kRaPlanThreads) {
    int before = -1, g = p.n_groups - 1;  // the first group whose items reach beyond it
    while (g - before > 1) {
      const int at = (before + g) >> 1;
      if (upto[at] <= i) before = at;
      else g = at;
    }
    const int steps = steps_of(-lens[g]), n = shared_parts((uint32_t)steps, prefix_part, p.prefix_parts), each = (steps + n - 1) / n;
    const uint32_t at = i - (g ? upto[g - 1] : 0), tile = at / (uint32_t)n;
    const int part = (int)(at - tile * (uint32_t)n);
    p.listed[i] = RaListedItem{group_q0[g], group_rows[g], (int)tile * kRaTileRows, 0, 0, -lens[g], g, 0, min(part * each, steps), min((part + 1) * each, steps), part, 0};
  }
  // ---- the items of the streams: those of a workgroup, then those of a wave, the longest of each first
  uint32_t singles = 0, waves = 0;
  if (tid < 64) {
    static_assert(kRaSizes == 64, "a lane to a size");
    const uint32_t single = sizes[lane], wave = sizes[kRaSizes + lane], singles_upto = sum_upto(single), waves_upto = sum_upto(wave);
    singles = of_lane(singles_upto, 63);
    waves = of_lane(waves_upto, 63);
    sizes[lane] = prefix_items + singles_upto - single;
    sizes[kRaSizes + lane] = prefix_items + singles + waves_upto - wave;
    if (lane == 0) {  // no more than there is room for, whatever the starts are
      const uint32_t heads_of = (uint32_t)p.kv_heads;
      *p.list = RaList{prefix_items * heads_of, min(prefix_items + singles, p.most_listed) * heads_of, min(prefix_items + singles + waves, p.most_listed) * heads_of, wide_own,
                       narrow_own};
    }
  }
  __syncthreads();
  for (int b0 = 0; b0 < p.streams; b0 += at_once) {
    const RaSharedStream s = stream(b0);
    each_tile(s, [&](int tile, int by_wave, int size, int steps, int parts, int part, float) {
      const uint32_t at = atomicAdd(&sizes[by_wave * kRaSizes + size], (uint32_t)parts);
      for (int i = 0; i < parts && at + i < p.most_listed; ++i)
        p.listed[at + i] = RaListedItem{s.q0, s.rows, tile * kRaTileRows, s.len, s.base, s.prefix_len, max(s.shares, 0), b0 + mine, min(i * part, steps), min((i + 1) * part, steps),
                                        s.joined || parts > 1 ? (int)p.prefix_parts + i : -1, 0};
    });
  }
}

// Joins, row by row, the parts of what a group attended together with the parts of the streams' own keys, and the parts of tiles that were cut:
// D / 4 lanes a row, the heads of one token to a workgroup, or some of them.
template <typename T, int D>
__global__ __launch_bounds__(kRaThreads) void shared_join_kernel(RaParams p) {
  constexpr int kRows = kRaThreads * 4 / D;
  const int lane = threadIdx.x & 63, column = threadIdx.x % (D / 4) * 4;
  const RaList list = *p.list;
  for (int64_t token = blockIdx.x; token < p.n_queries; token += gridDim.x) {
    // the last stream that begins at or before the token: 64 of what is left at a time
    int b = 0, left = p.streams + 1;
    while (left > 1) {
      const int step = (left + 63) / 64, at = lane * step;
      const int before = __popcll(__builtin_amdgcn_ballot_w64(at < left && p.q_starts[min(b + at, p.streams)] <= token));
      const int found = max(before - 1, 0) * step;
      b += found;
      left = min(step, left - found);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    if (b >= p.streams || p.q_starts[b] > token) continue;
    const RaSharedStream s = shared_stream(p, b);
    const RaJoined with = p.joined[b];
    for (int head = blockIdx.y * kRows + threadIdx.x / (D / 4); head < p.heads; head += gridDim.y * kRows) {
      const int f = (int)(token - s.q0) * (int)p.group.d + (int)((uint32_t)head - (uint32_t)head / p.group * p.group.d);
      const int steps = with.ahead + own_steps_of(p, s, min(f / kRaTileRows * kRaTileRows + kRaTileRows, s.rows) - 1);
      const int parts = shared_parts((uint32_t)steps, s.rows <= 32 ? list.narrow_part : list.wide_part, p.own_parts);
      if (!with.joined && parts <= 1) continue;  // its results are where they belong
      float m = -INFINITY, l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
      for (int i = 0; i < with.parts + parts; ++i) {
        const uint32_t slot = i < with.parts ? i : p.prefix_parts + i - with.parts;
        const float2 e = *shared_sums<D>(p, slot, token, head);
        const float4 y = *reinterpret_cast<const float4*>(shared_record<D>(p, slot, token, head) + column);
        const float top = fmaxf(m, e.x);
        const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * reference_unit<T>(p.scale_log2));
        const float c = e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((e.x - top) * reference_unit<T>(p.scale_log2));
        l = (m == -INFINITY ? l : l * a) + (e.x == -INFINITY ? e.y : e.y * c);  // as in the other joining launch
        v[0] = fmaf(y.x, c, v[0] * a);
        v[1] = fmaf(y.y, c, v[1] * a);
        v[2] = fmaf(y.z, c, v[2] * a);
        v[3] = fmaf(y.w, c, v[3] * a);
        m = top;
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      *reinterpret_cast<uint2*>(p.out + token * p.out_stride_token + head * p.out_stride_head + column) =
          make_uint2(T::pack2(v[0] * inv, v[1] * inv), T::pack2(v[2] * inv, v[3] * inv));
    }
  }
}

static int check_ragged(const ll_ragged_attention_args* a) {
  LL_REQUIRE(a, "ll_ragged_attention: no arguments");
  LL_REQUIRE(a->dtype == LL_DTYPE_BF16 || a->dtype == LL_DTYPE_F16, "ll_ragged_attention: dtype %d is not bf16 or f16", a->dtype);
  LL_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "ll_ragged_attention: head_dim %d is not 64 or 128", a->head_dim);
  LL_REQUIRE(a->num_kv_heads > 0 && a->num_heads > 0 && a->num_heads % a->num_kv_heads == 0 && a->num_heads <= 65536,
             "ll_ragged_attention: %d heads over %d kv heads", a->num_heads, a->num_kv_heads);
  LL_REQUIRE(a->n_queries >= 0 && a->streams >= 0, "ll_ragged_attention: %lld queries in %lld streams", (long long)a->n_queries, (long long)a->streams);
  LL_REQUIRE(a->n_queries <= 0x7fffffffll / a->num_heads, "ll_ragged_attention: %lld queries of %d heads are more than 2^31 rows",
             (long long)a->n_queries, a->num_heads);
  LL_REQUIRE(a->streams <= 0xfffffff / a->num_kv_heads, "ll_ragged_attention: %lld streams", (long long)a->streams);
  LL_REQUIRE(a->softmax_scale > 0.0f && std::isfinite(a->softmax_scale * kLog2E), "ll_ragged_attention: softmax_scale has to be positive");
  LL_REQUIRE(a->max_q_len >= 0 && a->max_kv_len >= 0, "ll_ragged_attention: negative longest lengths");
  if (a->page_table || a->page_size) {
    LL_REQUIRE(a->page_size > 0 && a->table_width >= 0 && a->n_pages >= 0 && a->n_pages <= 0x7fffffffll,
               "ll_ragged_attention: %lld pages of %d rows, tables of %lld", (long long)a->n_pages, a->page_size, (long long)a->table_width);
    LL_REQUIRE(a->table_width <= 0x7fffffffll / a->page_size, "ll_ragged_attention: a table of %lld pages of %d rows reaches beyond 2^31 keys",
               (long long)a->table_width, a->page_size);
    LL_REQUIRE(a->window >= 0 && a->sink_keys >= 0, "ll_ragged_attention: negative window or kept keys");
  } else {
    LL_REQUIRE(!a->causal && a->window == 0, "ll_ragged_attention: order and windows are for paged keys");
    LL_REQUIRE(a->n_keys >= 0 && a->n_keys <= 0x7fffffffll, "ll_ragged_attention: %lld keys", (long long)a->n_keys);
  }
  return LL_OK;
}

// How a launch is divided (host arithmetic): as many workgroups as the device holds, and the steps of a part.  Only the device knows
// the streams' lengths; the host knows the longest, if it is told, and how many rows there are in all.
// Parts make items alike and cost a record each, written and read: 66 KB for a tile of 128 rows of 128 columns, 15 us of a workgroup's share
// of the memory's rate.  us by steps of a part, 12 streams of 1 to 700 tokens x 40 heads over 300 to 9000 keys: 10 241, 16 200, 24 183, 48
// 176, whole tiles 256 (the rule: 56); 17 streams of 3 to 900 x 20 over 100 to 2400 masked states: 10 61, 16 74, 24 and more 85 (the rule:
// 11).  Narrow tiles, 32 single tokens x 32 heads over 500 to 16384 keys: 8 135, 12 130, 16 123, 24 132, 32 126 (the rule: 16); 4 over
// 4000: 8 20.4, 16 23.6, 32 34.3 (the rule: 8).
// Where tiles are alike, the number of parts follows from their cost, in sixteenths of a step of a full unit: steps are faster by themselves
// (kRaStepCost), an item's beginning and a record are paid for by the share of the device that they keep busy.  us by steps of a part, one
// stream of 100 x 32 / 8 heads of 128 columns over 1000 keys: 3 22.6, 4 23.2, 6 23.7, 8 27.6, whole 30.9 (the rule: 4); over 4000: 6 37.9, 8
// 31.8, 10 33.9, 16 38.8 (8); 500 x 12 heads of 64 over 9500: 10 47.4, 16 44.3, 24 53.1 (15); 532 x 40 / 8 over 9000 in pages of 24: 20 170, 47
// 143 (47).
struct RaPlan {
  uint32_t groups, part_steps, narrow_part_steps, records;
  size_t bytes;
  float part_share;
};
constexpr int64_t kRaStepCost[2][3] = {{9, 12, 16}, {12, 16, 16}};  // 64 and 128 columns: with one, two or three workgroups to a unit
constexpr int64_t kRaItemCost = 48, kRaRecordCost = 109;            // of items as many as the device holds: their beginnings, their records
constexpr int64_t kRaJoinCost = 40;                                 // of the second launch
constexpr int64_t kRaLeastNarrowSteps = 8, kRaMostNarrowSteps = 16, kRaMostWholeSteps = 32;
// Of what a workgroup has to do in all, a part: by the device, of up to 64 streams, where the launch is not so long that the last items do not
// count.  us with 0.5 / 0.75 / 0.9 / 1.1 / by the host's guess, pages for eight times the streams' keys: 12 streams of 1 to 700 tokens x 40 / 8
// heads over 300 to 9000 keys 207 / 216 / 204 / 199 / 274; 16 of 5 to 600 x 24 over 600 to 4600 173 / 176 / 173 / 173 / 196; 30 of 1 to 300 x
// 32 / 8 over 300 to 4000 97 / 99 / 89 / 96 / 100; prompts of 5 times 100 to 2000 x 16 / 4, causal, 82 / 101 / 84 / 83 / 74 (there whole; 74
// also with 0.9 and the records that the plan has for them).
constexpr float kRaShare = 0.9f;
constexpr int64_t kRaNarrowJoin = 7;                                // of the second launch behind narrow tiles, in their steps
constexpr size_t kRaMostBytes = (size_t)256 << 20;  // of records

static RaPlan plan_ragged(const ll_ragged_attention_args& a, int cus) {
  RaPlan r{0, 0, 0, 0, 0, 0.0f};
  if (a.n_queries == 0 || a.streams == 0) return r;
  const bool paged = a.page_table || a.page_size;
  const int64_t group = a.num_heads / a.num_kv_heads, slots = (a.head_dim == 64 ? 3 : 2) * cus;
  const int64_t longest = a.max_q_len > 0 && a.max_q_len < a.n_queries ? a.max_q_len : a.n_queries;
  const int64_t tiles = std::min(a.n_queries * group / kRaTileRows + a.streams, a.streams * ((longest * group + kRaTileRows - 1) / kRaTileRows));
  const int64_t all_keys = paged ? a.table_width * a.page_size : a.n_keys, rows_of_keys = paged ? std::min<int64_t>(a.n_pages * a.page_size, 1ll << 60) : a.n_keys;
  int64_t keys = a.max_kv_len > 0 && a.max_kv_len < all_keys ? a.max_kv_len : all_keys;
  bool alike = a.streams == 1;  // whether all tiles see about as many keys
  if (a.window > 0 && a.window < keys && a.sink_keys < keys) {
    // Without causal order a tile sees from its window's beginning to the last key.  Of several streams only the windows count all the same:
    // parts of the longer tiles cost more than they save, 3 of 900 to 2640 x 12 heads of 128 columns over 5000 to 13200 keys, window 1024, 117
    // us, so cut 148; 9 of 100 to 2640 x 8 of 64, window 512, 67 and 80.  A single stream, 2640 x 4 of 128 over 13200 keys: by the window alone
    // 48 us (1024) and 68 (64), by all that is seen 41 and 39; 1500 x 16 of 64 over 9000, window 2000, 70 and 74; 2640 x 24 of 128, 4096, 215 and 216.
    const int64_t seen = a.window + a.sink_keys + (a.causal || a.streams > 1 ? kRaTileRows / group : longest) + kRaKeys;
    alike = alike || 2 * seen < keys;
    keys = std::min(keys, seen);
  }
  const int64_t steps = std::max<int64_t>((keys + kRaKeys - 1) / kRaKeys, 1), busy = tiles * a.num_kv_heads;
  // Narrow tiles are bound by memory: parts short enough to keep the device busy to the end whatever the lengths are.
  r.narrow_part_steps = (uint32_t)std::min(std::max((steps * busy + 4 * slots - 1) / (4 * slots), kRaLeastNarrowSteps), kRaMostNarrowSteps);
  // As alike count tiles too few to fill half of the device, whose longest ones decide, and streams in a cache with room for long ones alone.
  const int64_t room = a.streams * keys;
  if (alike || 2 * busy <= cus || (5 * rows_of_keys >= 4 * room && 4 * rows_of_keys <= 5 * room)) {
    int64_t best = 1, least = -1;
    for (int64_t parts = 1; parts <= 64 && (parts == 1 || steps / parts >= 3); ++parts) {
      const int64_t each = (steps + parts - 1) / parts, items = busy * parts, rounds = (items + slots - 1) / slots;
      const int64_t step = kRaStepCost[a.head_dim == 128][items <= cus ? 0 : items <= 2 * cus ? 1 : 2];
      const int64_t cost = rounds * (each * step + kRaItemCost * std::min(items, slots) / slots) + (parts > 1 ? kRaJoinCost + kRaRecordCost * items / slots : 0);
      if (least < 0 || cost < least) {
        least = cost;
        best = parts;
      }
    }
    r.part_steps = best == 1 ? 1u << 24 : (uint32_t)((steps + best - 1) / best);
  } else if (steps <= 16) {  // 12 x 20 to 300 tokens x 16 heads of 64 columns over 300 to 1000 keys whole 24.2 us, by 10 steps 26.4
    r.part_steps = 1u << 24;
  } else {  // about what a workgroup has to do in all (kRaShare), or if the mean stream has half of the keys that there is room for
    const int64_t mean = std::min(steps, (rows_of_keys / a.streams + kRaKeys - 1) / kRaKeys + 1) / 2 + 1;
    r.part_steps = (uint32_t)std::min<int64_t>(std::max<int64_t>(busy * mean * 5 / (4 * slots), kRaLeastWideSteps), 1 << 24);
    if (a.streams <= 64 && busy <= 8 * slots) r.part_share = kRaShare * a.num_kv_heads / slots;
  }
  const bool all_narrow = longest * group <= 32;
  // Beside wider tiles, streams of few rows are worth a second launch only where they are long.  By themselves, where the steps that they
  // save, one behind the other, are more than the second launch costs; the memory serves half as many items as there are units at full pace,
  // more of them take as long cut or whole.  us whole / cut, single tokens: 8 streams x 16 heads of 64 columns over 640 keys 8.7 / 11.2, over
  // 1280 12.7 / 15.7; 1 x 8 of 128 over 640 12.4 / 13.9, over 1024 16.9 / 15.4; 32 x 8 of 128 over 100 to 1024 19.4 / 22.0, to 1600 26.0 / 24.7,
  // to 2048 30.9 / 32.5.
  const int64_t served = 2 * busy * steps / cus;
  if (all_narrow ? steps <= kRaMostWholeSteps && std::max(steps, served) <= kRaNarrowJoin + std::max(kRaLeastNarrowSteps, served)
                 : a.streams == 1 || steps <= 2 * kRaMostNarrowSteps)
    r.narrow_part_steps = 1u << 24;
  const int64_t part = all_narrow ? r.narrow_part_steps : std::min(r.part_steps, r.narrow_part_steps);
  const int64_t parts = r.part_share != 0.0f && !all_narrow ? (steps + kRaLeastWideSteps - 1) / kRaLeastWideSteps : (steps + part - 1) / part;
  if (parts > 1) {
    // Every tile in as many parts, or what is allowed; streams that find no records left stay whole.
    const size_t record = 32 * (size_t)(a.head_dim + 2) * sizeof(float);
    int64_t want = tiles * parts * (all_narrow ? 1 : kRaTileRows / 32);
    // Parts as many as the share makes, and one more of every tile.  Of causal prompts, whose tiles see up to twice their mean, all parts may be
    // more; streams that find no records left stay whole.  us so / with records for every part: prompts of 5 times 100 to 2000 x 16 / 4 heads
    // of 128 columns 74 / 83, 2 of 300 to 4000 x 16 / 4 of 64 77 / 93, 4 of 50 to 2000 tokens x 16 / 4 over 700 to 3000 keys 81 / 86, 2 of
    // 2000 x 8 / 2 75 / 66.
    if (r.part_share != 0.0f && !all_narrow)
      want = std::min(want, (int64_t)((1.0f / r.part_share + 1 + tiles) * (kRaTileRows / 32)) + a.streams * ((steps + r.narrow_part_steps - 1) / r.narrow_part_steps));
    r.records = (uint32_t)std::min<int64_t>(want, (int64_t)(kRaMostBytes / record) / a.num_kv_heads);
    r.bytes = r.records * record * a.num_kv_heads;
  }
  const int64_t items = (a.n_queries * group / kRaTileRows + a.streams) * a.num_kv_heads * (r.records ? parts : 1);
  r.groups = (uint32_t)std::min(slots, items);
  return r;
}

}  // namespace ll

extern "C" int ll_ragged_attention_workspace(const ll_ragged_attention_args* a, int compute_units, size_t* bytes) {
  using namespace ll;
  if (int rc = check_ragged(a)) return rc;
  LL_REQUIRE(bytes && compute_units >= 0, "ll_ragged_attention_workspace: nowhere to put the answer");
  if (compute_units == 0) {
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev)) {
      set_error("ll_ragged_attention_workspace: hipGetDevice failed: %s", hipGetErrorString(e));
      return LL_ELAUNCH;
    }
    if (int rc = compute_units_of(dev, compute_units, "ll_ragged_attention_workspace")) return rc;
  }
  *bytes = plan_ragged(*a, compute_units).bytes;
  return LL_OK;
}

namespace ll {
template <typename T, int D, int KIND>
static int launch_ragged(const RaParams& p, uint32_t grid, hipStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  const void* kernel = reinterpret_cast<const void*>(&ragged_attention_kernel<T, D, KIND>);
  if (int rc = allow_dynamic_lds(kernel, kRaLds<D>, allowed, "ll_ragged_attention")) return rc;
  ragged_attention_kernel<T, D, KIND><<<grid, kRaThreads, kRaLds<D>, stream>>>(p);
  LL_CHECK_LAUNCH("ll_ragged_attention");
  if (p.records) {
    const uint32_t each = kRaThreads * 4 / D;
    ragged_join_kernel<T, D, KIND><<<dim3(kRaJoinGroups, kRaTileRows / each / 2), kRaThreads, 0, stream>>>(p);
    LL_CHECK_LAUNCH("ll_ragged_attention (join)");
  }
  return LL_OK;
}
template <typename T, int D>
static int launch_ragged(const RaParams& p, int kind, uint32_t grid, hipStream_t stream) {
  if (kind == kRaPaged) return launch_ragged<T, D, kRaPaged>(p, grid, stream);
  if (kind == kRaRows) return launch_ragged<T, D, kRaRows>(p, grid, stream);
  return launch_ragged<T, D, kRaMaskedRows>(p, grid, stream);
}

static int check_ragged_pointers(const ll_ragged_attention_args* a) {
  const bool paged = a->page_table || a->page_size;
  const bool has_keys = paged ? a->n_pages > 0 && a->table_width > 0 : a->n_keys > 0;
  LL_REQUIRE(a->q && a->out, "ll_ragged_attention: null q or out");
  LL_REQUIRE(a->streams == 0 || (a->q_starts && (paged ? a->kv_lens && (a->page_table || a->table_width == 0) : a->k_starts != nullptr)),
             "ll_ragged_attention: null starts, lengths or page table");
  LL_REQUIRE(!has_keys || (a->k && a->v), "ll_ragged_attention: null k or v");
  LL_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->k | (uintptr_t)a->v) % 16 == 0,
             "ll_ragged_attention: q, k, v and out must be 16-byte aligned");
  LL_REQUIRE((a->q_stride_token | a->q_stride_head | a->out_stride_token | a->out_stride_head | a->k_stride_page | a->k_stride_row |
              a->k_stride_head | a->v_stride_page | a->v_stride_row | a->v_stride_head) % 8 == 0,
             "ll_ragged_attention: strides must be multiples of 8 elements");
  LL_REQUIRE(a->k_stride_page >= 0 && a->v_stride_page >= 0 && a->k_stride_page <= 0xffffffffll && a->v_stride_page <= 0xffffffffll &&
                 a->k_stride_row >= 0 && a->v_stride_row >= 0 && a->k_stride_row < (1ll << 26) && a->v_stride_row < (1ll << 26),
             "ll_ragged_attention: pages of k and v lie at most 2^32 elements apart, rows 2^26");
  return LL_OK;
}

static RaParams ragged_params(const ll_ragged_attention_args* a) {
  const bool paged = a->page_table || a->page_size;
  const bool has_keys = paged ? a->n_pages > 0 && a->table_width > 0 : a->n_keys > 0;
  RaParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.out = static_cast<uint16_t*>(a->out);
  p.q_stride_token = a->q_stride_token;
  p.q_stride_head = a->q_stride_head;
  p.out_stride_token = a->out_stride_token;
  p.out_stride_head = a->out_stride_head;
  p.n_queries = a->n_queries;
  p.streams = (int)a->streams;
  p.q_starts = a->q_starts;
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.k_stride_page = (uint32_t)a->k_stride_page;
  p.k_stride_row = (uint32_t)a->k_stride_row;
  p.k_stride_head = a->k_stride_head;
  p.v_stride_page = (uint32_t)a->v_stride_page;
  p.v_stride_row = (uint32_t)a->v_stride_row;
  p.v_stride_head = a->v_stride_head;
  p.page_table = a->page_table;
  p.table_stride = a->table_stride;
  p.table_keys = paged && has_keys ? a->table_width * a->page_size : 0;
  p.n_pages = (uint32_t)a->n_pages;
  p.page = divisor(paged ? (uint32_t)a->page_size : 1u);
  p.kv_lens = a->kv_lens;
  p.k_starts = a->k_starts;
  p.k_lens = a->k_lens;
  p.key_mask = a->key_mask;
  p.n_keys = a->n_keys;
  p.scale_log2 = a->softmax_scale * kLog2E;
  p.causal = a->causal;
  p.heads = a->num_heads;
  p.kv_heads = a->num_kv_heads;
  p.group = divisor((uint32_t)(a->num_heads / a->num_kv_heads));
  p.window = (uint32_t)std::min<int64_t>(a->window, 0x7fffffff);  // keys are fewer
  p.sink = (uint32_t)std::min<int64_t>(a->sink_keys, 0x7fffffff);
  return p;
}
}  // namespace ll

extern "C" int ll_ragged_attention(const ll_ragged_attention_args* a, void* stream) {
  using namespace ll;
  if (int rc = check_ragged(a)) return rc;
  if (a->n_queries == 0) return LL_OK;
  if (int rc = check_ragged_pointers(a)) return rc;
  int dev = 0, cus = 0;
  if (hipError_t e = hipGetDevice(&dev)) {
    set_error("ll_ragged_attention: hipGetDevice failed: %s", hipGetErrorString(e));
    return LL_ELAUNCH;
  }
  if (int rc = compute_units_of(dev, cus, "ll_ragged_attention")) return rc;
  const RaPlan plan = plan_ragged(*a, cus);
  LL_REQUIRE(plan.bytes == 0 || (a->workspace && (uintptr_t)a->workspace % 16 == 0 && a->workspace_bytes >= plan.bytes),
             "ll_ragged_attention: a workspace of %zu bytes, 16-byte aligned, is needed", plan.bytes);
  RaParams p = ragged_params(a);
  p.groups = plan.groups;
  p.part_steps = plan.part_steps;
  p.part_share = plan.part_share;
  p.narrow_part_steps = plan.narrow_part_steps;
  p.records = plan.records;
  p.record_mem = static_cast<float*>(a->workspace);
  const uint32_t grid = p.groups + (a->clear_rest ? kRaClearGroups : 0);
  if (grid == 0) return LL_OK;
  const bool paged = a->page_table || a->page_size;
  const int kind = paged ? kRaPaged : a->key_mask ? kRaMaskedRows : kRaRows;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == LL_DTYPE_BF16)
    return a->head_dim == 128 ? launch_ragged<Bf16, 128>(p, kind, grid, s) : launch_ragged<Bf16, 64>(p, kind, grid, s);
  return a->head_dim == 128 ? launch_ragged<F16, 128>(p, kind, grid, s) : launch_ragged<F16, 64>(p, kind, grid, s);
}

namespace ll {
static int check_shared(const ll_shared_prefix_args* a) {
  LL_REQUIRE(a, "ll_shared_prefix_attention: no arguments");
  if (int rc = check_ragged(&a->own)) return rc;
  LL_REQUIRE(a->own.page_size > 0, "ll_shared_prefix_attention: keys lie in pages");
  LL_REQUIRE(a->own.window == 0 && a->own.sink_keys == 0, "ll_shared_prefix_attention: there are no windows");
  LL_REQUIRE(a->groups >= 0 && a->groups <= 0xfffffff, "ll_shared_prefix_attention: %lld groups", (long long)a->groups);
  LL_REQUIRE(a->max_prefix_len >= 0, "ll_shared_prefix_attention: negative longest beginning");
  LL_REQUIRE(a->prefix_width >= 0 && a->prefix_width <= (1ll << 30) / a->own.page_size && a->own.table_width <= (1ll << 30) / a->own.page_size,
             "ll_shared_prefix_attention: tables of %lld and %lld pages of %d rows reach beyond 2^30 keys", (long long)a->prefix_width,
             (long long)a->own.table_width, a->own.page_size);
  return LL_OK;
}

// How a launch over shared beginnings is divided (host arithmetic).  Without parts of beginnings every stream goes over its group's by itself,
// divided as keys of one table are.
struct SharedPlan {
  RaPlan alone;
  uint32_t groups, prefix_parts, own_parts;  // parts of a tile at most: the device makes as many as fit
  uint32_t most_listed;
  size_t list, listed, joined, bytes;  // where they begin in the workspace, behind the records; all of it
};
constexpr size_t kRaMostSharedBytes = (size_t)256 << 20;  // of records, where there are more than two of a row
constexpr int64_t kRaMostParts = 64;
// What a launch to list the items and one to join their results have to save, in steps of all workgroups: some 10 us.  Steps of narrow tiles
// are shorter.  A group takes as long as so many steps more, for its tile's beginning, for its records, and since keys that its streams go over one
// after the other come from the caches but for the first time.  us joined / direct on the one side, single tokens x 24 heads of 128 columns: 16
// streams over 1000 keys 25.5 / 26.3, over 2000 26 / 58, 16 groups of 4 over 2000 112 / 195, 4 over 4000 28 / 33, 16 of 33 to 64 tokens over 2000 57 /
// 82; on the other: 16 over 500 22.6 / 19.3, 16 groups of 4 over 500 58 / 52, 16 of 4 x 32 / 8 heads over 1000 39 / 28, 4 x 32 / 8 over 4000 25 / 20,
// 16 of 33 to 64 tokens x 12 of 64 over 2000 35 / 32.  Wrong by most: 4 of 33 to 64 tokens x 16 / 4 heads of 64 over 2000 stay direct, 27 / 56.
constexpr int64_t kRaJoinedSteps = 5, kRaJoinedNarrowSteps = 7, kRaJoinedGroupSteps = 20;

// A stream's keys and those of its group's beginning as if they were in one table.
static ll_ragged_attention_args one_table(const ll_shared_prefix_args& s) {
  ll_ragged_attention_args a = s.own;
  const int64_t own = a.table_width * a.page_size, shared = s.groups ? s.prefix_width * a.page_size : 0;
  const auto told = [](int64_t n, int64_t reach) { return n > 0 && n < reach ? n : reach; };
  a.max_kv_len = told(a.max_kv_len, own) + told(s.max_prefix_len, shared);
  a.table_width += s.groups ? s.prefix_width : 0;
  return a;
}

static SharedPlan plan_shared(const ll_shared_prefix_args& s, int cus) {
  const ll_ragged_attention_args& a = s.own;
  SharedPlan r{};
  r.own_parts = 1;
  if (a.n_queries == 0 || a.streams == 0) return r;
  const int64_t group = a.num_heads / a.num_kv_heads, slots = (a.head_dim == 64 ? 3 : 2) * cus;
  const int64_t longest = a.max_q_len > 0 && a.max_q_len < a.n_queries ? a.max_q_len : a.n_queries;
  const int64_t streams = std::min(a.streams, a.n_queries);  // with rows
  const int64_t tiles = std::min(a.n_queries * group / kRaTileRows + streams, streams * ((longest * group + kRaTileRows - 1) / kRaTileRows));
  const auto steps_within = [&](int64_t told, int64_t width) {
    const int64_t reach = width * a.page_size, keys = told > 0 && told < reach ? told : reach;
    return (keys + kRaKeys - 1) / kRaKeys;
  };
  const int64_t own_steps = steps_within(a.max_kv_len, a.n_pages ? a.table_width : 0);
  const int64_t prefix_steps = s.groups && a.n_pages ? steps_within(s.max_prefix_len, s.prefix_width) : 0;
  const int64_t groups = std::min(s.groups, streams), together = a.n_queries * group / kRaTileRows + groups;  // tiles of whole groups
  const size_t rows = (size_t)a.n_queries * a.num_heads, part_bytes = rows * (a.head_dim + 2) * sizeof(float);
  // The second line: groups of which, on average, none comes near being joined (4 x 2640 tokens x 24 heads over 10560 + 2640 keys).
  if (streams > 1 && s.groups <= kRaJoinedGroups && part_bytes <= 4 * kRaMostSharedBytes &&
      streams * prefix_steps >= kRaJoinedCost / 2 * together &&
      ((tiles - together) * prefix_steps - kRaJoinedGroupSteps * groups) * a.num_kv_heads > (longest * group <= 32 ? kRaJoinedNarrowSteps : kRaJoinedSteps) * slots) {
    // No tile has more parts than there are workgroups for each head, since a workgroup's share is not below that much of one tile.
    const int64_t most = std::max<int64_t>(std::min<int64_t>(kRaMostParts, (int64_t)(kRaMostSharedBytes / part_bytes)), 2);
    // of streams whose group is not joined, over its beginning too: 16 groups of some 4 single tokens, a few of one, x 24 heads over 4000 keys 187 us;
    // without 322
    r.own_parts = (uint32_t)std::max<int64_t>(std::min<int64_t>((own_steps + prefix_steps + kRaLeastOwnPart - 1) / kRaLeastOwnPart, most / 4), 1);
    r.prefix_parts = (uint32_t)std::min(std::min<int64_t>((prefix_steps + kRaLeastPrefixPart - 1) / kRaLeastPrefixPart, slots / a.num_kv_heads + 1), most - r.own_parts);
    const int64_t items = together * r.prefix_parts + (a.n_queries * group / kRaTileRows + streams) * r.own_parts;
    r.groups = (uint32_t)std::min(slots, items * a.num_kv_heads);
    r.most_listed = (uint32_t)std::min<int64_t>(items, 0xffffffffll / a.num_kv_heads);
    const auto behind = [](size_t bytes) { return (bytes + 63) / 64 * 64; };
    r.list = behind(part_bytes * (r.prefix_parts + r.own_parts));
    r.listed = behind(r.list + sizeof(RaList));
    r.joined = behind(r.listed + items * sizeof(RaListedItem));
    r.bytes = r.joined + a.streams * sizeof(RaJoined);
  } else {
    r.alone = plan_ragged(one_table(s), cus);
    r.groups = r.alone.groups;
    r.bytes = r.alone.bytes;
  }
  return r;
}

template <typename T, int D>
static int launch_shared(const RaParams& p, uint32_t grid, uint32_t units, hipStream_t stream) {
  if (p.prefix_parts == 0) return launch_ragged<T, D, kRaPrefixed>(p, grid, stream);
  static std::atomic<uint64_t> allowed{0};
  constexpr size_t kLds = kRaLds<D>;
  const void* kernel = reinterpret_cast<const void*>(&ragged_attention_kernel<T, D, kRaListed>);
  if (int rc = allow_dynamic_lds(kernel, kLds, allowed, "ll_shared_prefix_attention")) return rc;
  shared_plan_kernel<D><<<1, kRaPlanThreads, 0, stream>>>(p, units);
  LL_CHECK_LAUNCH("ll_shared_prefix_attention (items)");
  ragged_attention_kernel<T, D, kRaListed><<<grid, kRaThreads, kLds, stream>>>(p);
  LL_CHECK_LAUNCH("ll_shared_prefix_attention");
  const uint32_t rows = kRaThreads * 4 / D;
  const dim3 join((uint32_t)std::min<int64_t>(p.n_queries, 4096), ((uint32_t)p.heads + rows - 1) / rows);
  shared_join_kernel<T, D><<<join, kRaThreads, 0, stream>>>(p);
  LL_CHECK_LAUNCH("ll_shared_prefix_attention (join)");
  return LL_OK;
}
}  // namespace ll

extern "C" int ll_shared_prefix_attention_workspace(const ll_shared_prefix_args* a, int compute_units, size_t* bytes) {
  using namespace ll;
  if (int rc = check_shared(a)) return rc;
  LL_REQUIRE(bytes && compute_units >= 0, "ll_shared_prefix_attention_workspace: nowhere to put the answer");
  if (compute_units == 0) {
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev)) {
      set_error("ll_shared_prefix_attention_workspace: hipGetDevice failed: %s", hipGetErrorString(e));
      return LL_ELAUNCH;
    }
    if (int rc = compute_units_of(dev, compute_units, "ll_shared_prefix_attention_workspace")) return rc;
  }
  *bytes = plan_shared(*a, compute_units).bytes;
  return LL_OK;
}

extern "C" int ll_shared_prefix_attention(const ll_shared_prefix_args* args, void* stream) {
  using namespace ll;
  if (int rc = check_shared(args)) return rc;
  const ll_ragged_attention_args* a = &args->own;
  if (a->n_queries == 0) return LL_OK;
  if (int rc = check_ragged_pointers(a)) return rc;
  const bool shares = args->groups > 0 && args->prefix_width > 0 && a->n_pages > 0;
  LL_REQUIRE(!shares || (args->prefix_lens && args->prefix_table), "ll_shared_prefix_attention: null lengths or table of what is shared");
  LL_REQUIRE(args->groups <= 1 || args->group_starts, "ll_shared_prefix_attention: %lld groups without their beginnings", (long long)args->groups);
  LL_REQUIRE(!shares || (a->k && a->v), "ll_shared_prefix_attention: null k or v");
  int dev = 0, cus = 0;
  if (hipError_t e = hipGetDevice(&dev)) {
    set_error("ll_shared_prefix_attention: hipGetDevice failed: %s", hipGetErrorString(e));
    return LL_ELAUNCH;
  }
  if (int rc = compute_units_of(dev, cus, "ll_shared_prefix_attention")) return rc;
  const SharedPlan plan = plan_shared(*args, cus);
  LL_REQUIRE(plan.bytes == 0 || (a->workspace && (uintptr_t)a->workspace % 16 == 0 && a->workspace_bytes >= plan.bytes),
             "ll_shared_prefix_attention: a workspace of %zu bytes, 16-byte aligned, is needed", plan.bytes);
  RaParams p = ragged_params(a);
  p.groups = plan.groups;
  p.part_steps = plan.alone.part_steps;
  p.part_share = plan.alone.part_share;
  p.narrow_part_steps = plan.alone.narrow_part_steps;
  p.records = plan.alone.records;
  p.prefix_parts = plan.prefix_parts;
  p.own_parts = plan.own_parts;
  p.record_mem = static_cast<float*>(a->workspace);
  if (plan.prefix_parts) {
    uint8_t* const memory = static_cast<uint8_t*>(a->workspace);
    p.list = reinterpret_cast<RaList*>(memory + plan.list);
    p.listed = reinterpret_cast<RaListedItem*>(memory + plan.listed);
    p.most_listed = plan.most_listed;
    p.joined = reinterpret_cast<RaJoined*>(memory + plan.joined);
  }
  p.n_groups = shares ? (int)args->groups : 0;
  p.group_starts = args->group_starts;
  p.prefix_lens = args->prefix_lens;
  p.prefix_table = args->prefix_table;
  p.prefix_stride = args->prefix_stride;
  p.prefix_keys = shares ? args->prefix_width * a->page_size : 0;
  const uint32_t grid = p.groups + (a->clear_rest ? kRaClearGroups : 0);
  if (grid == 0) return LL_OK;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->dtype == LL_DTYPE_BF16) return a->head_dim == 128 ? launch_shared<Bf16, 128>(p, grid, cus, st) : launch_shared<Bf16, 64>(p, grid, cus, st);
  return a->head_dim == 128 ? launch_shared<F16, 128>(p, grid, cus, st) : launch_shared<F16, 64>(p, grid, cus, st);
}
