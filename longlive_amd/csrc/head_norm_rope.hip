// Every head of q and k of a batch of tokens through its own RMS norm and the position rotation, K and V on to the rows of a
// paged cache, in one pass (ll_head_norm_rope).
//
//   y = x * rsqrt(mean(x^2) + eps) * w over a head's D columns;  (a, b) -> (a cos - b sin, b cos + a sin) over pairs of columns
//
// D / 8 lanes hold a head, rounded up to 8, 16 or 32, eight columns each, as two groups of four that are each other's partners
// in the rotation: 4 l and 4 l + R / 2 for pairs of halves, 8 l and 8 l + 4 for neighbouring pairs (and for columns that are not
// rotated).  Either way pair j of lane l is j = 4 l .. 4 l + 3, so that the angles are one load of 16 bytes each and nothing
// passes between lanes but the sum of squares.
#include "ll_types16.h"

namespace ll {

struct HeadRows {
  const uint16_t* x;
  uint16_t* out;
  const void* weight;
  int64_t stride_token, stride_head, out_stride_token, out_stride_head;
  int heads, weight_f32;
};

struct HeadNormParams {
  HeadRows rows[3];  // q, k, v
  int64_t first_token;
  uint32_t tokens;       // of this launch
  uint32_t units_q, units_kv;  // units of kHeads heads: q's, and k's (and v's)
  Divisor per_token;
  int D, R, interleaved;
  float eps, inv_D;
  const float *cos, *sin;
  int64_t table_rows;
  const int64_t *positions, *slots;
  int64_t n_slots;
};

// Sum over LANES neighbouring lanes, in every one of them.
template <int LANES>
__device__ __forceinline__ float sum_over_lanes(float v) {
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) v += __shfl_xor(v, d);
  return v;
}

template <typename T>
__device__ __forceinline__ void load4(const uint16_t* p, float* f) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  T::unpack2(w.x, f[0], f[1]);
  T::unpack2(w.y, f[2], f[3]);
}

constexpr int kHeadNormThreads = 256;

// LANES hold a head; a group of them takes HEADS heads of one token, one behind the other.
template <typename T, int LANES, int HEADS>
__global__ __launch_bounds__(kHeadNormThreads) void head_norm_rope_kernel(HeadNormParams p) {
  const uint32_t unit = blockIdx.x * (kHeadNormThreads / LANES) + threadIdx.x / LANES;
  const uint32_t local = unit / p.per_token;
  if (local >= p.tokens) return;  // uniform over a group
  uint32_t at = unit - local * p.per_token.d;
  const int64_t t = p.first_token + local;
  const int l = threadIdx.x % LANES;
  const bool active = l * 8 < p.D;
  int kind = 0;
  if (at >= p.units_q) {
    at -= p.units_q;
    kind = 1;
    if (at >= p.units_kv) {
      at -= p.units_kv;
      kind = 2;
    }
  }
  const HeadRows& r = p.rows[kind];
  const bool halves = !p.interleaved && 8 * l < p.R;
  const int c0 = halves ? 4 * l : 8 * l, c1 = halves ? 4 * l + p.R / 2 : 8 * l + 4;
  int64_t row = t;
  if (kind != 0 && p.slots) {
    row = p.slots[t];
    if ((uint64_t)row >= (uint64_t)p.n_slots) return;
  }
  float cs[4] = {1.0f, 1.0f, 1.0f, 1.0f}, sn[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t pos = p.positions ? p.positions[t] : t;
  const bool rotate = kind != 2 && 8 * l < p.R && (uint64_t)pos < (uint64_t)p.table_rows;
  if (rotate) {
    const int64_t a = pos * (p.R / 2) + 4 * l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cs[i] = p.cos[a + i];
      sn[i] = p.sin[a + i];
    }
  }
  float w[8];
  if (r.weight && active) {
    if (r.weight_f32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = static_cast<const float*>(r.weight)[c0 + i];
        w[4 + i] = static_cast<const float*>(r.weight)[c1 + i];
      }
    } else {
      load4<T>(static_cast<const uint16_t*>(r.weight) + c0, w);
      load4<T>(static_cast<const uint16_t*>(r.weight) + c1, w + 4);
    }
  }
  for (int i = 0; i < HEADS; ++i) {
    const int h = at * HEADS + i;
    if (h >= r.heads) return;
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    const uint16_t* src = r.x + t * r.stride_token + h * r.stride_head;
    if (active) {
      load4<T>(src + c0, x);
      load4<T>(src + c1, x + 4);
    }
    if (r.weight) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
      const float scale = rsqrtf(fmaf(sum_over_lanes<LANES>(sum), p.inv_D, p.eps));
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * scale * w[j];
    }
    if (rotate) {
      if (halves) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = x[j], b = x[4 + j];
          x[j] = a * cs[j] - b * sn[j];
          x[4 + j] = b * cs[j] + a * sn[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = x[2 * j], b = x[2 * j + 1];
          x[2 * j] = a * cs[j] - b * sn[j];
          x[2 * j + 1] = b * cs[j] + a * sn[j];
        }
      }
    }
    uint16_t* dst = r.out + row * r.out_stride_token + h * r.out_stride_head;
    if (active) {
      *reinterpret_cast<uint2*>(dst + c0) = make_uint2(T::pack2(x[0], x[1]), T::pack2(x[2], x[3]));
      *reinterpret_cast<uint2*>(dst + c1) = make_uint2(T::pack2(x[4], x[5]), T::pack2(x[6], x[7]));
    }
  }
}

template <typename T, int LANES>
void launch_head_norm(const HeadNormParams& p, uint32_t units, hipStream_t stream) {
  const uint32_t per_wg = kHeadNormThreads / LANES;
  head_norm_rope_kernel<T, LANES, 1><<<(units + per_wg - 1) / per_wg, kHeadNormThreads, 0, stream>>>(p);
}

static int check_rows(const ll_head_rows* r, const char* name, bool may_norm) {
  LL_REQUIRE(r, "ll_head_norm_rope: %s is NULL", name);
  LL_REQUIRE(r->num_heads >= 0 && r->num_heads <= 65536, "ll_head_norm_rope: %s has %d heads", name, r->num_heads);
  if (r->num_heads == 0) return LL_OK;
  LL_REQUIRE(r->x && r->out, "ll_head_norm_rope: null pointer in %s", name);
  LL_REQUIRE(((uintptr_t)r->x | (uintptr_t)r->out | (uintptr_t)r->weight) % 16 == 0, "ll_head_norm_rope: pointers of %s must be 16-byte aligned", name);
  LL_REQUIRE((r->stride_token | r->stride_head | r->out_stride_token | r->out_stride_head) % 8 == 0,
             "ll_head_norm_rope: strides of %s must be multiples of 8", name);
  LL_REQUIRE(may_norm || !r->weight, "ll_head_norm_rope: %s has no norm", name);
  return LL_OK;
}

}  // namespace ll

extern "C" int ll_head_norm_rope(int dtype, int64_t tokens, int head_dim, const ll_head_rows* q, const ll_head_rows* k, const ll_head_rows* v,
                                 float eps, const float* cos, const float* sin, int64_t table_rows, int rotary_dim, const int64_t* positions,
                                 int interleaved, const int64_t* slots, int64_t n_slots, void* stream) {
  using namespace ll;
  LL_REQUIRE(dtype == LL_DTYPE_BF16 || dtype == LL_DTYPE_F16, "ll_head_norm_rope: dtype %d is not bf16 or f16", dtype);
  LL_REQUIRE(tokens >= 0 && tokens < (1ll << 40), "ll_head_norm_rope: %lld tokens", (long long)tokens);
  LL_REQUIRE(head_dim > 0 && head_dim <= 256 && head_dim % 8 == 0, "ll_head_norm_rope: head_dim %d is not a multiple of 8 up to 256", head_dim);
  LL_REQUIRE(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 8 == 0,
             "ll_head_norm_rope: rotary_dim %d is not a multiple of 8 up to head_dim %d", rotary_dim, head_dim);
  LL_REQUIRE(rotary_dim == 0 || (cos && sin && table_rows >= 0), "ll_head_norm_rope: no angles to rotate by");
  LL_REQUIRE(((uintptr_t)cos | (uintptr_t)sin) % 16 == 0, "ll_head_norm_rope: cos and sin must be 16-byte aligned");
  const ll_head_rows none{};
  if (!v) v = &none;
  if (int rc = check_rows(q, "q", true)) return rc;
  if (int rc = check_rows(k, "k", true)) return rc;
  if (int rc = check_rows(v, "v", false)) return rc;
  LL_REQUIRE(v->num_heads == 0 || (slots && v->num_heads == k->num_heads), "ll_head_norm_rope: v goes with slots and has as many heads as k");
  LL_REQUIRE(!slots || n_slots >= 0, "ll_head_norm_rope: %lld slots", (long long)n_slots);
  HeadNormParams p{};
  const ll_head_rows* given[3] = {q, k, v};
  for (int i = 0; i < 3; ++i) {
    const ll_head_rows& r = *given[i];
    p.rows[i] = HeadRows{static_cast<const uint16_t*>(r.x), static_cast<uint16_t*>(r.out), r.weight, r.stride_token, r.stride_head,
                         r.out_stride_token, r.out_stride_head, r.num_heads, r.weight_f32};
  }
  p.D = head_dim;
  p.R = rotary_dim;
  p.interleaved = interleaved;
  p.eps = eps;
  p.inv_D = 1.0f / (float)head_dim;
  p.cos = cos;
  p.sin = sin;
  p.table_rows = table_rows;
  p.positions = positions;
  p.slots = slots;
  p.n_slots = n_slots;
  p.units_q = (uint32_t)q->num_heads;
  p.units_kv = (uint32_t)k->num_heads;
  const uint32_t per_token = p.units_q + p.units_kv + (uint32_t)v->num_heads;
  if (per_token == 0 || tokens == 0) return LL_OK;
  p.per_token = divisor(per_token);
  const int64_t most = (1ll << 30) / per_token;  // units are numbered in 32 bits
  for (int64_t first = 0; first < tokens; first += most) {
    p.first_token = first;
    p.tokens = (uint32_t)(tokens - first < most ? tokens - first : most);
    const uint32_t units = p.tokens * per_token;
    const hipStream_t s = static_cast<hipStream_t>(stream);
#define LL_LAUNCH(T)                                            \
  if (head_dim <= 64) {                                         \
    launch_head_norm<T, 8>(p, units, s);                        \
  } else if (head_dim <= 128) {                                 \
    launch_head_norm<T, 16>(p, units, s);                       \
  } else {                                                      \
    launch_head_norm<T, 32>(p, units, s);                       \
  }
    if (dtype == LL_DTYPE_BF16) {
      LL_LAUNCH(Bf16)
    } else {
      LL_LAUNCH(F16)
    }
#undef LL_LAUNCH
    LL_CHECK_LAUNCH("ll_head_norm_rope");
  }
  return LL_OK;
}
