// Attention of a batch of streams of different length (ll_ragged_attention): new tokens over the keys of a paged cache, or
// queries over encoder states whose number differs from stream to stream.
//
//   out[t, h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale * (q[t, h] . k_j - max)),   j over the keys that row t may see
//
// The rows of a kv head's queries, (token, head of the group) one behind the other, are cut into tiles of 128.  A workgroup of
// four waves walks the keys of a tile 64 at a time: K and V come into LDS, every wave multiplies them with its own 32 rows,
//   S^T = K Q^T  and  O^T = V^T P^T   (v_mfma_f32_32x32x16),
// so that a lane owns one row: its maximum and sum need one exchange between the wave's halves, its mask two comparisons per
// score with bounds of its own, and its rescaling is a multiplication by a scalar.  The probabilities leave the first product in
// the registers in which the second one wants them, keys permuted; V^T is read permuted alike by the LDS read that transposes.
#include "ll_types16.h"

#include <cmath>

namespace ll {

constexpr int kRaThreads = 256;
constexpr int kRaTileRows = 128;  // rows of a workgroup, 32 a wave
constexpr int kRaKeys = 64;       // keys of a step
constexpr int kRaClearGroups = 16;

struct RaParams {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_stride_token, q_stride_head, out_stride_token, out_stride_head;
  int64_t n_queries, streams;
  const int32_t* q_starts;
  const uint16_t *k, *v;
  int64_t k_stride_page, k_stride_row, k_stride_head, v_stride_page, v_stride_row, v_stride_head;
  const int32_t* page_table;
  int64_t table_stride, table_keys;  // keys that a stream's row of the table reaches
  uint32_t n_pages;
  Divisor page;
  const int32_t *kv_lens, *k_starts, *k_lens;
  const uint8_t* key_mask;
  int64_t n_keys;
  float scale_log2;
  int causal, clear_rest;
  int heads, kv_heads;
  Divisor group;       // heads of a kv head
  int64_t window, sink;
  uint32_t tiles;      // workgroups of a (stream, kv head); each takes every tiles-th tile
  uint32_t work_groups;
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

// The keys of a stream.
struct Keys {
  int64_t len;              // keys 0 .. len - 1
  int64_t start;            // ragged: row of key 0
  const int32_t* pages;     // paged: the stream's row of the table
};

// Whether key j exists and, if so, its row's offset in K and V.
template <bool PAGED>
__device__ __forceinline__ bool find_key(const RaParams& p, const Keys& keys, int64_t j, int64_t& k_at, int64_t& v_at) {
  if (j < 0 || j >= keys.len) return false;
  if constexpr (PAGED) {
    const uint32_t page = (uint32_t)j / p.page, row = (uint32_t)j - page * p.page.d;
    const uint32_t entry = (uint32_t)keys.pages[page];
    if (entry >= p.n_pages) return false;
    k_at = (int64_t)entry * p.k_stride_page + row * p.k_stride_row;
    v_at = (int64_t)entry * p.v_stride_page + row * p.v_stride_row;
  } else {
    const int64_t row = keys.start + j;
    if (p.key_mask && p.key_mask[row] == 0) return false;
    k_at = row * p.k_stride_row;
    v_at = row * p.v_stride_row;
  }
  return true;
}

template <typename T, int D, bool PAGED>
__global__ __launch_bounds__(kRaThreads) void ragged_attention_kernel(RaParams p) {
  constexpr int kRowBytes = 2 * D, kPieces = D / 8, kDTiles = D / 32, kSteps = D / 16;
  __shared__ __attribute__((aligned(16))) uint8_t k_lds[kRaKeys * kRowBytes];
  __shared__ __attribute__((aligned(16))) uint8_t v_lds[kRaKeys * kRowBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, lh = lane >> 5;
  auto start_of = [&](int64_t b) { return min(max((int64_t)p.q_starts[b], (int64_t)0), p.n_queries); };

  if (blockIdx.x >= p.work_groups) {  // rows outside every stream
    const int64_t first = p.streams ? start_of(0) : 0, end = p.streams ? max(start_of(p.streams), first) : 0;
    const int64_t outside = first + p.n_queries - end, pieces = outside * p.heads * kPieces;
    for (int64_t i = (int64_t)(blockIdx.x - p.work_groups) * kRaThreads + tid; i < pieces; i += (int64_t)kRaClearGroups * kRaThreads) {
      const int64_t row = i / (p.heads * kPieces);
      const int at = (int)(i - row * (p.heads * kPieces)), h = at / kPieces, c = at % kPieces;
      uint16_t* dst = p.out + (row < first ? row : row - first + end) * p.out_stride_token + h * p.out_stride_head + 8 * c;
      *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
    }
    return;
  }

  const uint32_t pair = blockIdx.x / p.tiles, hk = pair % p.kv_heads;
  const int64_t b = pair / p.kv_heads;
  const int64_t q0 = start_of(b), n = max(start_of(b + 1) - q0, (int64_t)0), rows = n * p.group.d;
  Keys keys{};
  if constexpr (PAGED) {
    keys.len = min(max((int64_t)p.kv_lens[b], (int64_t)0), p.table_keys);
    keys.pages = p.page_table + b * p.table_stride;
  } else {
    keys.start = min(max((int64_t)p.k_starts[b], (int64_t)0), p.n_keys);
    const int64_t len = p.k_lens ? (int64_t)p.k_lens[b] : (int64_t)p.k_starts[b + 1] - keys.start;
    keys.len = min(max(len, (int64_t)0), p.n_keys - keys.start);
  }
  const uint16_t *k_head = p.k + hk * p.k_stride_head, *v_head = p.v + hk * p.v_stride_head;

  for (int64_t tile = blockIdx.x % p.tiles; tile * kRaTileRows < rows; tile += p.tiles) {
    const int64_t f0 = tile * kRaTileRows, f1 = min(f0 + kRaTileRows, rows) - 1;
    // this lane's row
    const int64_t f = min(f0 + wave * 32 + l32, rows - 1);
    const int64_t i = (uint32_t)f / p.group, pos = keys.len - n + i;
    const int head = hk * p.group.d + (int)(f - i * p.group.d);
    short8v qf[kSteps];
    {
      const uint16_t* src = p.q + (q0 + i) * p.q_stride_token + head * p.q_stride_head + 8 * lh;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) qf[ks] = *reinterpret_cast<const short8v*>(src + 16 * ks);
    }
    // Keys that the row sees: those below `last`, from `from` on or below `sink`.
    const int64_t pos0 = keys.len - n + (uint32_t)f0 / p.group, pos1 = keys.len - n + (uint32_t)f1 / p.group;
    const int64_t last = p.causal ? min(pos + 1, keys.len) : keys.len;
    const int64_t from = p.window ? max(pos - p.window + 1, (int64_t)0) : 0;
    const int64_t last0 = p.causal ? min(pos0 + 1, keys.len) : keys.len, last1 = p.causal ? min(pos1 + 1, keys.len) : keys.len;
    const int64_t from0 = p.window ? max(pos0 - p.window + 1, (int64_t)0) : 0, from1 = p.window ? max(pos1 - p.window + 1, (int64_t)0) : 0;
    // Steps of 64 keys: those with kept first keys, then those from the first row's window on.
    const int64_t end_step = max((last1 + kRaKeys - 1) / kRaKeys, (int64_t)0), from_step = from0 / kRaKeys;
    const int64_t sink_steps = min((min(p.sink, from0) + kRaKeys - 1) / kRaKeys, from_step);
    const int64_t n_steps = min(sink_steps, end_step) + max(end_step - from_step, (int64_t)0);

    float16v o[kDTiles];
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    for (int64_t s = 0; s < n_steps; ++s) {
      const int64_t base = (s < sink_steps ? s : from_step + s - sink_steps) * kRaKeys;
      __syncthreads();
#pragma unroll
      for (int it = 0; it < kRaKeys * kPieces / kRaThreads; ++it) {
        const int row = (it * kRaThreads + tid) / kPieces, c = tid % kPieces;
        int64_t k_at, v_at;
        uint4 kv = make_uint4(0, 0, 0, 0), vv = make_uint4(0, 0, 0, 0);
        if (find_key<PAGED>(p, keys, base + row, k_at, v_at)) {
          kv = *reinterpret_cast<const uint4*>(k_head + k_at + 8 * c);
          vv = *reinterpret_cast<const uint4*>(v_head + v_at + 8 * c);
        }
        *reinterpret_cast<uint4*>(k_lds + row * kRowBytes + k_piece<D>(row, c) * 16) = kv;
        *reinterpret_cast<uint4*>(v_lds + row * kRowBytes + v_piece<D>(row, c) * 16) = vv;
      }
      int64_t k_at, v_at;
      const uint64_t there = __builtin_amdgcn_ballot_w64(find_key<PAGED>(p, keys, base + lane, k_at, v_at));
      __syncthreads();

      // S^T: register r of sc[kt] is key 32 kt + 8 (r / 4) + 4 lh + r % 4
      float16v sc[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[kt][r] = 0.0f;
        const int row = 32 * kt + l32;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
          const short8v a = *reinterpret_cast<const short8v*>(k_lds + row * kRowBytes + k_piece<D>(row, 2 * ks + lh) * 16);
          sc[kt] = T::mfma(a, qf[ks], sc[kt]);
        }
      }
      const bool all_seen = there == ~0ull && base + kRaKeys <= last0 && (base >= from1 || base + kRaKeys <= p.sink);
      if (!all_seen) {
        const uint64_t bits = there >> (4 * lh);
        const int64_t first = base + 4 * lh;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int at = 32 * kt + 8 * (r / 4) + r % 4;
            const int64_t key = first + at;
            const bool seen = key < last && (key >= from || key < p.sink) && ((bits >> at) & 1);
            sc[kt][r] = seen ? sc[kt][r] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[kt][r]);
      mx = fmaxf(exchange_max(mx), m);
      // a row that has seen nothing yet stays at -inf; 0 stands for it in the exponents, where -inf - -inf would be NaN
      const float neg = mx == -INFINITY ? 0.0f : -mx * p.scale_log2;
      const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaf(m, p.scale_log2, neg));
      m = mx;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        uint32_t w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[step >> 1][8 * (step & 1) + 2 * u], p.scale_log2, neg));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[step >> 1][8 * (step & 1) + 2 * u + 1], p.scale_log2, neg));
          l += p0 + p1;
          w[u] = T::pack2(p0, p1);
        }
        const short8v pb = __builtin_bit_cast(short8v, make_uint4(w[0], w[1], w[2], w[3]));
        typedef __attribute__((address_space(3))) short4v* lds_short4;
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt) {
          short4v part[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int row = 16 * step + 8 * j + 4 * lh + ((lane & 15) >> 2);
            const int piece = 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)(v_lds + row * kRowBytes + v_piece<D>(row, piece) * 16 + (lane & 1) * 8));
          }
          o[dt] = T::mfma(__builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7), pb, o[dt]);
        }
      }
    }
    l = exchange_sum(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (f0 + wave * 32 + l32 < rows) {
      uint16_t* dst = p.out + (q0 + i) * p.out_stride_token + head * p.out_stride_head + 4 * lh;
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<uint2*>(dst + 32 * dt + 8 * g) =
              make_uint2(T::pack2(o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv), T::pack2(o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv));
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
  LL_REQUIRE(a->streams <= 0x7fffffffll / a->num_kv_heads - 64, "ll_ragged_attention: %lld streams", (long long)a->streams);
  LL_REQUIRE(a->softmax_scale > 0.0f && std::isfinite(a->softmax_scale), "ll_ragged_attention: softmax_scale has to be positive");
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

}  // namespace ll

extern "C" int ll_ragged_attention_workspace(const ll_ragged_attention_args* a, int compute_units, size_t* bytes) {
  using namespace ll;
  if (int rc = check_ragged(a)) return rc;
  LL_REQUIRE(bytes && compute_units >= 0, "ll_ragged_attention_workspace: nowhere to put the answer");
  *bytes = 0;
  return LL_OK;
}

extern "C" int ll_ragged_attention(const ll_ragged_attention_args* a, void* stream) {
  using namespace ll;
  if (int rc = check_ragged(a)) return rc;
  if (a->n_queries == 0) return LL_OK;
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
  RaParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.out = static_cast<uint16_t*>(a->out);
  p.q_stride_token = a->q_stride_token;
  p.q_stride_head = a->q_stride_head;
  p.out_stride_token = a->out_stride_token;
  p.out_stride_head = a->out_stride_head;
  p.n_queries = a->n_queries;
  p.streams = a->streams;
  p.q_starts = a->q_starts;
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.k_stride_page = a->k_stride_page;
  p.k_stride_row = a->k_stride_row;
  p.k_stride_head = a->k_stride_head;
  p.v_stride_page = a->v_stride_page;
  p.v_stride_row = a->v_stride_row;
  p.v_stride_head = a->v_stride_head;
  p.page_table = a->page_table;
  p.table_stride = a->table_stride;
  p.table_keys = paged ? a->table_width * a->page_size : 0;
  p.n_pages = (uint32_t)a->n_pages;
  p.page = divisor(paged ? (uint32_t)a->page_size : 1u);
  p.kv_lens = a->kv_lens;
  p.k_starts = a->k_starts;
  p.k_lens = a->k_lens;
  p.key_mask = a->key_mask;
  p.n_keys = a->n_keys;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.causal = a->causal;
  p.clear_rest = a->clear_rest;
  p.heads = a->num_heads;
  p.kv_heads = a->num_kv_heads;
  p.group = divisor((uint32_t)(a->num_heads / a->num_kv_heads));
  p.window = a->window;
  p.sink = a->sink_keys;
  const int64_t longest = a->max_q_len > 0 && a->max_q_len < a->n_queries ? a->max_q_len : a->n_queries;
  int64_t tiles = (longest * p.group.d + kRaTileRows - 1) / kRaTileRows;
  const int64_t pairs = a->streams * a->num_kv_heads;
  if (pairs > 0 && tiles > 0x3fffffffll / pairs) tiles = 0x3fffffffll / pairs > 0 ? 0x3fffffffll / pairs : 1;
  p.tiles = (uint32_t)tiles;
  p.work_groups = (uint32_t)(pairs * tiles);
  const uint32_t grid = p.work_groups + (a->clear_rest ? kRaClearGroups : 0);
  if (grid == 0) return LL_OK;
  const hipStream_t s = static_cast<hipStream_t>(stream);
#define LL_LAUNCH(T, D)                                                                             \
  if (paged) {                                                                                      \
    ragged_attention_kernel<T, D, true><<<grid, kRaThreads, 0, s>>>(p);                             \
  } else {                                                                                          \
    ragged_attention_kernel<T, D, false><<<grid, kRaThreads, 0, s>>>(p);                            \
  }
  if (a->dtype == LL_DTYPE_BF16) {
    if (a->head_dim == 128) {
      LL_LAUNCH(Bf16, 128)
    } else {
      LL_LAUNCH(Bf16, 64)
    }
  } else {
    if (a->head_dim == 128) {
      LL_LAUNCH(F16, 128)
    } else {
      LL_LAUNCH(F16, 64)
    }
  }
#undef LL_LAUNCH
  LL_CHECK_LAUNCH("ll_ragged_attention");
  return LL_OK;
}
