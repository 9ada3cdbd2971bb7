// Every head of q and k of a batch of tokens through its own RMS norm and the position rotation, K and V on to the rows of a
// paged cache, in one pass (ll_head_norm_rope).
//
//   y = x * rsqrt(mean(x^2) + eps) * w over a head's D columns;  (a, b) -> (a cos - b sin, b cos + a sin) over pairs of columns
//
// D / 8 lanes hold a head, rounded up to 8, 16 or 32, eight columns each, as two groups of four that are each other's partners
// in the rotation: 4 l and 4 l + R / 2 for pairs of halves, 8 l and 8 l + 4 for neighbouring pairs (and for columns that are not
// rotated).  Either way pair j of lane l is j = 4 l .. 4 l + 3, so that the angles are one load of 16 bytes each and nothing
// passes between lanes but the sum of squares.  A wave takes heads of one token and one of q, k and v: position, slot, pointers and
// strides are scalars, loaded once for up to two heads per lane, all of whose loads are under way before the first is used.  (With a wave
// across q, k and v, the pointers came per lane out of the argument segment, which lies in host memory: 2640 x (24 + 24) heads of 128 182 us.)
//
// Bound by memory: 2640 x (24 + 24) heads of 128 columns, 66 MB, 13.0 us, 5.1 TB/s (half of it out of the last-level cache when repeated);
// 16381 x (40 + 8 + 8) of 64, 237 MB, 53 us, 4.4 TB/s; 24 x (16 + 4 + 4), a decoding step, 3.3 us of the GPU, 5.6 us a call.
#include "head_norm_split.h"
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
  uint32_t tokens;             // of this launch
  uint32_t units_q, units_kv;  // waves per token for q, and for k (and v)
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
  if constexpr (LANES == 8) {
#define LL_DPP_ADD(v, ctrl) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xF, 0xF, true))
    LL_DPP_ADD(v, 0xB1);   // quad_perm [1, 0, 3, 2]
    LL_DPP_ADD(v, 0x4E);   // quad_perm [2, 3, 0, 1]
    LL_DPP_ADD(v, 0x141);  // row_half_mirror
#undef LL_DPP_ADD
    return v;
  } else {
    v = sum_over_16_lanes(v);
    return LANES == 16 ? v : v + __shfl_xor(v, 16);
  }
}

template <typename T>
__device__ __forceinline__ void unpack4(uint2 w, float* f) {
  T::unpack2(w.x, f[0], f[1]);
  T::unpack2(w.y, f[2], f[3]);
}

// Two heads a lane once the device has waves enough: us with one / two, 1000 tokens x (32 + 8 + 8) heads 8.6 / 9.0, 2640 x (24 + 24) 14.9 / 14.1,
// 16000 x (32 + 8 + 8) 92.9 / 72.4, 16381 x (40 + 8 + 8) of 64 columns 57.0 / 46.2 (four: 74.2 and 44.3).
constexpr int64_t kManyWaves = 8192;

// LANES hold a head, a wave 64 / LANES heads side by side, HEADS times.
template <typename T, int LANES, int HEADS>
__global__ __launch_bounds__(kHeadNormThreads) void head_norm_rope_kernel(HeadNormParams p) {
  constexpr int kSide = 64 / LANES;
  const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * (kHeadNormThreads / 64) + threadIdx.x / 64);
  const uint32_t local = unit / p.per_token;
  if (local >= p.tokens) return;
  uint32_t at = unit - local * p.per_token.d;
  const int64_t t = p.first_token + local;
  int kind = 0;
  if (at >= p.units_q) {
    at -= p.units_q;
    kind = 1;
    if (at >= p.units_kv) {
      at -= p.units_kv;
      kind = 2;
    }
  }
  kind = __builtin_amdgcn_readfirstlane(kind);
  const HeadRows r = p.rows[kind];
  int64_t row = t;
  if (kind != 0 && p.slots) {
    row = p.slots[t];
    if ((uint64_t)row >= (uint64_t)p.n_slots) return;
  }
  const int64_t pos = p.positions ? p.positions[t] : t;
  const int l = threadIdx.x % LANES, h0 = (int)at * kSide * HEADS + (int)(threadIdx.x & 63) / LANES;
  const bool active = l * 8 < p.D;
  const bool halves = !p.interleaved && 8 * l < p.R;
  const int c0 = halves ? 4 * l : 8 * l, c1 = halves ? 4 * l + p.R / 2 : 8 * l + 4;

  uint2 x[HEADS][2], w[2] = {};
  float4 wf[2] = {}, cs = make_float4(1.0f, 1.0f, 1.0f, 1.0f), sn = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const uint16_t* src = r.x + t * r.stride_token;
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = h0 + i * kSide;
    if (active && h < r.heads) {
      x[i][0] = *reinterpret_cast<const uint2*>(src + h * r.stride_head + c0);
      x[i][1] = *reinterpret_cast<const uint2*>(src + h * r.stride_head + c1);
    } else {
      x[i][0] = x[i][1] = make_uint2(0, 0);
    }
  }
  if (r.weight && active) {
    if (r.weight_f32) {
      wf[0] = *reinterpret_cast<const float4*>(static_cast<const float*>(r.weight) + c0);
      wf[1] = *reinterpret_cast<const float4*>(static_cast<const float*>(r.weight) + c1);
    } else {
      w[0] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(r.weight) + c0);
      w[1] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(r.weight) + c1);
    }
  }
  const bool rotate = kind != 2 && p.R != 0 && (uint64_t)pos < (uint64_t)p.table_rows;
  if (rotate && 8 * l < p.R) {
    cs = *reinterpret_cast<const float4*>(p.cos + pos * (p.R / 2) + 4 * l);
    sn = *reinterpret_cast<const float4*>(p.sin + pos * (p.R / 2) + 4 * l);
  }
  float f[8] = {wf[0].x, wf[0].y, wf[0].z, wf[0].w, wf[1].x, wf[1].y, wf[1].z, wf[1].w};
  if (r.weight && !r.weight_f32) {
    unpack4<T>(w[0], f);
    unpack4<T>(w[1], f + 4);
  }
  const float cc[4] = {cs.x, cs.y, cs.z, cs.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
  uint16_t* dst = r.out + row * r.out_stride_token;
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = h0 + i * kSide;
    float y[8];
    unpack4<T>(x[i][0], y);
    unpack4<T>(x[i][1], y + 4);
    if (r.weight) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(y[j], y[j], sum);
      const float scale = rsqrtf(fmaf(sum_over_lanes<LANES>(sum), p.inv_D, p.eps));
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = y[j] * scale * f[j];
    }
    if (rotate && 8 * l < p.R) {
      const bool apart = halves;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = apart ? y[j] : y[2 * j], b = apart ? y[4 + j] : y[2 * j + 1];
        const float a2 = a * cc[j] - b * ss[j], b2 = b * cc[j] + a * ss[j];
        if (apart) {
          y[j] = a2;
          y[4 + j] = b2;
        } else {
          y[2 * j] = a2;
          y[2 * j + 1] = b2;
        }
      }
    }
    if (active && h < r.heads) {
      *reinterpret_cast<uint2*>(dst + h * r.out_stride_head + c0) = make_uint2(T::pack2(y[0], y[1]), T::pack2(y[2], y[3]));
      *reinterpret_cast<uint2*>(dst + h * r.out_stride_head + c1) = make_uint2(T::pack2(y[4], y[5]), T::pack2(y[6], y[7]));
    }
  }
}

// Waves of LANES lanes a head and `heads` heads a lane that a token takes.
static uint32_t waves_for(int num_heads, int lanes, int heads) {
  const int each = 64 / lanes * heads;
  return (uint32_t)((num_heads + each - 1) / each);
}

template <typename T, int LANES, int HEADS>
static void launch_head_norm(HeadNormParams p, int64_t tokens, hipStream_t stream) {
  p.units_q = waves_for(p.rows[0].heads, LANES, HEADS);
  p.units_kv = waves_for(p.rows[1].heads, LANES, HEADS);
  const uint32_t per_token = p.units_q + p.units_kv + waves_for(p.rows[2].heads, LANES, HEADS);
  p.per_token = divisor(per_token);
  const int64_t most = head_norm_tokens(per_token);
  for (int64_t first = 0; first < tokens; first += most) {
    p.first_token = first;
    p.tokens = (uint32_t)(tokens - first < most ? tokens - first : most);
    head_norm_rope_kernel<T, LANES, HEADS><<<head_norm_groups(p.tokens, per_token), kHeadNormThreads, 0, stream>>>(p);
  }
}

template <typename T, int LANES>
static void launch_head_norm(const HeadNormParams& p, int64_t tokens, hipStream_t stream) {
  const int64_t waves = tokens * (waves_for(p.rows[0].heads, LANES, 1) + 2 * waves_for(p.rows[1].heads, LANES, 1));
  if (waves > kManyWaves)
    launch_head_norm<T, LANES, 2>(p, tokens, stream);
  else
    launch_head_norm<T, LANES, 1>(p, tokens, stream);
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
  if (tokens == 0 || q->num_heads + k->num_heads == 0) return LL_OK;
  const hipStream_t s = static_cast<hipStream_t>(stream);
#define LL_LAUNCH(T)                           \
  if (head_dim <= 64) {                        \
    launch_head_norm<T, 8>(p, tokens, s);      \
  } else if (head_dim <= 128) {                \
    launch_head_norm<T, 16>(p, tokens, s);     \
  } else {                                     \
    launch_head_norm<T, 32>(p, tokens, s);     \
  }
  if (dtype == LL_DTYPE_BF16) {
    LL_LAUNCH(Bf16)
  } else {
    LL_LAUNCH(F16)
  }
#undef LL_LAUNCH
  LL_CHECK_LAUNCH("ll_head_norm_rope");
  return LL_OK;
}
