// Every head of q and k of a batch of tokens through its own RMS norm and the position rotation, K and V on to the rows of a
// paged cache, in one pass: by angles from a table (ll_head_norm_rope) or formed from positions and frequencies (ll_rotate_by_position).
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

#include <cmath>

namespace ll {

struct HeadRows {
  const uint16_t* x;
  uint16_t* out;
  const void* weight;
  int64_t stride_token, stride_head, out_stride_token, out_stride_head;
  int heads, weight_f32;
};

// Angles formed in the kernel.
struct FormedAngles {
  const double* frequencies;
  float amplitude;
  Divisor frame, columns;    // tokens of a video frame and of a row in it; 0: positions on a line
  int frame_pairs, row_pairs;  // pairs turned by frames, by rows; the others by columns
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
  FormedAngles formed;
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
// With angles formed it depends on where the rows come from.  Out of memory: 2000 x (32 + 8 + 8) 14.5 / 14.1, 2640 x (24 + 24) 16.2 / 15.1 (of video frames
// 16.2 / 16.1), 10560 x (24 + 24) 50.1 / 46.2 (50.9 / 47.1), 10560 x (32 + 8) 41.3 / 39.7, 16381 x (40 + 8 + 8) of 64 columns 51.0 / 50.7, 40000 x (32 + 8 + 8)
// 190 / 182.  Where one call repeats another and finds its rows in the last-level cache, one head may be a little faster: 2640 x (24 + 24) 13.0 / 13.5 (13.5 /
// 14.3), 10560 x (32 + 8) 33.3 / 34.4, 16381 x (40 + 8 + 8) 35.8 / 37.8, but not 2000 x (32 + 8 + 8) 9.9 / 8.8 nor 10560 x (24 + 24) 42.9 / 41.8.  The rule goes
// by the former.
constexpr int64_t kManyWaves = 8192;

// Cosines and sines of pairs 4 l .. 4 l + 3 at a position, which is the wave's.  A position times a frequency takes 64 bits: at position
// 2^20 its rounding to 32 would turn the fastest pairs by 2^-4.  The matter is settled in turns, of which the whole ones are dropped; what is
// left is exact to 2^-26 of a turn in 32 bits, and the hardware's sine and cosine of it
// are off by no more than 2^-22, a thousandth of the rounding to f16 that follows.
// Formed once for the wave's heads, it hides behind their loads: 40000 x (32 + 8 + 8) heads of 128 columns, 983 MB, 176 us, 5.6 TB/s; 16381 x (40 + 8
// + 8) of 64 with 32 rotated, 235 MB, 49, and 36 out of the last-level cache; 2640 x (24 + 24) by video frames, 65 MB, 14.1, without the table's 90 MB for 176 000
// positions; 24 x (16 + 4 + 4) 3.4 on the device, 5.6 from call to call.
__device__ __forceinline__ void form_angles(const FormedAngles& a, int64_t pos, int l, float (&cs)[4], float (&sn)[4]) {
  double f[4];
  *reinterpret_cast<double2*>(f) = *reinterpret_cast<const double2*>(a.frequencies + 4 * l);
  *reinterpret_cast<double2*>(f + 2) = *reinterpret_cast<const double2*>(a.frequencies + 4 * l + 2);
  double at[3] = {(double)pos, 0.0, 0.0};
  if (a.frame.d) {
    int64_t frame;
    uint32_t in_frame;
    if ((uint64_t)pos >> 32 == 0) {
      frame = (uint32_t)pos / a.frame;
      in_frame = (uint32_t)pos - (uint32_t)frame * a.frame.d;
    } else {  // rounded down, also below zero
      frame = pos / (int64_t)a.frame.d;
      int64_t rest = pos - frame * a.frame.d;
      if (rest < 0) {
        rest += a.frame.d;
        --frame;
      }
      in_frame = (uint32_t)rest;
    }
    const uint32_t row = in_frame / a.columns;
    at[0] = (double)frame;
    at[1] = (double)row;
    at[2] = (double)(in_frame - row * a.columns.d);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int pair = 4 * l + j;
    const double x = !a.frame.d || pair < a.frame_pairs ? at[0] : pair < a.frame_pairs + a.row_pairs ? at[1] : at[2];
    const double turns = x * (f[j] * 0.15915494309189533577);  // 1 / (2 pi)
    const float part = (float)(turns - rint(turns));
    cs[j] = a.amplitude * __builtin_amdgcn_cosf(part);  // of a part of a turn
    sn[j] = a.amplitude * __builtin_amdgcn_sinf(part);
  }
}

// LANES hold a head, a wave 64 / LANES heads side by side, HEADS times.  FORMED: by angles formed from positions.
template <typename T, int LANES, int HEADS, bool FORMED>
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
  const bool rotate = kind != 2 && p.R != 0 && (FORMED || (uint64_t)pos < (uint64_t)p.table_rows);
  if (!FORMED && rotate && 8 * l < p.R) {
    cs = *reinterpret_cast<const float4*>(p.cos + pos * (p.R / 2) + 4 * l);
    sn = *reinterpret_cast<const float4*>(p.sin + pos * (p.R / 2) + 4 * l);
  }
  float f[8] = {wf[0].x, wf[0].y, wf[0].z, wf[0].w, wf[1].x, wf[1].y, wf[1].z, wf[1].w};
  if (r.weight && !r.weight_f32) {
    unpack4<T>(w[0], f);
    unpack4<T>(w[1], f + 4);
  }
  float cc[4] = {cs.x, cs.y, cs.z, cs.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
  if constexpr (FORMED) {
    if (rotate && 8 * l < p.R) form_angles(p.formed, pos, l, cc, ss);
  }
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

template <typename T, int LANES, int HEADS, bool FORMED>
static void launch_head_norm(HeadNormParams p, int64_t tokens, hipStream_t stream) {
  p.units_q = waves_for(p.rows[0].heads, LANES, HEADS);
  p.units_kv = waves_for(p.rows[1].heads, LANES, HEADS);
  const uint32_t per_token = p.units_q + p.units_kv + waves_for(p.rows[2].heads, LANES, HEADS);
  p.per_token = divisor(per_token);
  const int64_t most = head_norm_tokens(per_token);
  for (int64_t first = 0; first < tokens; first += most) {
    p.first_token = first;
    p.tokens = (uint32_t)(tokens - first < most ? tokens - first : most);
    head_norm_rope_kernel<T, LANES, HEADS, FORMED><<<head_norm_groups(p.tokens, per_token), kHeadNormThreads, 0, stream>>>(p);
  }
}

template <typename T, int LANES, bool FORMED>
static void launch_head_norm(const HeadNormParams& p, int64_t tokens, hipStream_t stream) {
  const int64_t waves = tokens * (waves_for(p.rows[0].heads, LANES, 1) + 2 * waves_for(p.rows[1].heads, LANES, 1));
  if (waves > kManyWaves)
    launch_head_norm<T, LANES, 2, FORMED>(p, tokens, stream);
  else
    launch_head_norm<T, LANES, 1, FORMED>(p, tokens, stream);
}

template <bool FORMED>
static void launch_head_norm(const HeadNormParams& p, int dtype, int64_t tokens, hipStream_t stream) {
#define LL_LAUNCH(T)                                   \
  if (p.D <= 64) {                                     \
    launch_head_norm<T, 8, FORMED>(p, tokens, stream);   \
  } else if (p.D <= 128) {                             \
    launch_head_norm<T, 16, FORMED>(p, tokens, stream);  \
  } else {                                             \
    launch_head_norm<T, 32, FORMED>(p, tokens, stream);  \
  }
  if (dtype == LL_DTYPE_BF16) {
    LL_LAUNCH(Bf16)
  } else {
    LL_LAUNCH(F16)
  }
#undef LL_LAUNCH
}

static int check_rows(const char* what, const ll_head_rows* r, const char* name, bool may_norm) {
  LL_REQUIRE(r, "%s: %s is NULL", what, name);
  LL_REQUIRE(r->num_heads >= 0 && r->num_heads <= 65536, "%s: %s has %d heads", what, name, r->num_heads);
  if (r->num_heads == 0) return LL_OK;
  LL_REQUIRE(r->x && r->out, "%s: null pointer in %s", what, name);
  LL_REQUIRE(((uintptr_t)r->x | (uintptr_t)r->out | (uintptr_t)r->weight) % 16 == 0, "%s: pointers of %s must be 16-byte aligned", what, name);
  LL_REQUIRE((r->stride_token | r->stride_head | r->out_stride_token | r->out_stride_head) % 8 == 0,
             "%s: strides of %s must be multiples of 8", what, name);
  LL_REQUIRE(may_norm || !r->weight, "%s: %s has no norm", what, name);
  return LL_OK;
}

// What both entry points take.
static int head_norm_params(const char* what, int dtype, int64_t tokens, int head_dim, const ll_head_rows* q, const ll_head_rows* k,
                            const ll_head_rows* v, float eps, int rotary_dim, const int64_t* positions, int interleaved, const int64_t* slots,
                            int64_t n_slots, HeadNormParams& p) {
  LL_REQUIRE(dtype == LL_DTYPE_BF16 || dtype == LL_DTYPE_F16, "%s: dtype %d is not bf16 or f16", what, dtype);
  LL_REQUIRE(tokens >= 0 && tokens < (1ll << 40), "%s: %lld tokens", what, (long long)tokens);
  LL_REQUIRE(head_dim > 0 && head_dim <= 256 && head_dim % 8 == 0, "%s: head_dim %d is not a multiple of 8 up to 256", what, head_dim);
  LL_REQUIRE(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 8 == 0,
             "%s: rotary_dim %d is not a multiple of 8 up to head_dim %d", what, rotary_dim, head_dim);
  const ll_head_rows none{};
  if (!v) v = &none;
  if (int rc = check_rows(what, q, "q", true)) return rc;
  if (int rc = check_rows(what, k, "k", true)) return rc;
  if (int rc = check_rows(what, v, "v", false)) return rc;
  LL_REQUIRE(v->num_heads == 0 || (slots && v->num_heads == k->num_heads), "%s: v goes with slots and has as many heads as k", what);
  LL_REQUIRE(!slots || n_slots >= 0, "%s: %lld slots", what, (long long)n_slots);
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
  p.positions = positions;
  p.slots = slots;
  p.n_slots = n_slots;
  return LL_OK;
}

}  // namespace ll

extern "C" int ll_head_norm_rope(int dtype, int64_t tokens, int head_dim, const ll_head_rows* q, const ll_head_rows* k, const ll_head_rows* v,
                                 float eps, const float* cos, const float* sin, int64_t table_rows, int rotary_dim, const int64_t* positions,
                                 int interleaved, const int64_t* slots, int64_t n_slots, void* stream) {
  using namespace ll;
  HeadNormParams p{};
  if (int rc = head_norm_params("ll_head_norm_rope", dtype, tokens, head_dim, q, k, v, eps, rotary_dim, positions, interleaved, slots, n_slots, p)) return rc;
  LL_REQUIRE(rotary_dim == 0 || (cos && sin && table_rows >= 0), "ll_head_norm_rope: no angles to rotate by");
  LL_REQUIRE(((uintptr_t)cos | (uintptr_t)sin) % 16 == 0, "ll_head_norm_rope: cos and sin must be 16-byte aligned");
  p.cos = cos;
  p.sin = sin;
  p.table_rows = table_rows;
  if (tokens == 0 || q->num_heads + k->num_heads == 0) return LL_OK;
  launch_head_norm<false>(p, dtype, tokens, static_cast<hipStream_t>(stream));
  LL_CHECK_LAUNCH("ll_head_norm_rope");
  return LL_OK;
}

extern "C" int ll_rotate_by_position(int dtype, int64_t tokens, int head_dim, const ll_head_rows* q, const ll_head_rows* k, const ll_head_rows* v,
                                     float eps, const ll_position_angles* angles, const int64_t* positions, int interleaved, const int64_t* slots,
                                     int64_t n_slots, void* stream) {
  using namespace ll;
  LL_REQUIRE(angles, "ll_rotate_by_position: no angles to rotate by");
  HeadNormParams p{};
  if (int rc = head_norm_params("ll_rotate_by_position", dtype, tokens, head_dim, q, k, v, eps, angles->rotary_dim, positions, interleaved, slots, n_slots, p))
    return rc;
  LL_REQUIRE(p.R == 0 || (angles->frequencies && (uintptr_t)angles->frequencies % 16 == 0), "ll_rotate_by_position: frequencies must be 16-byte aligned");
  LL_REQUIRE(std::isfinite(angles->amplitude), "ll_rotate_by_position: amplitude %g", (double)angles->amplitude);
  const int64_t rows = angles->grid_rows, columns = angles->grid_columns;
  LL_REQUIRE(rows >= 0 && columns >= 0 && (rows > 0) == (columns > 0) && rows <= 0x7fffffffll && columns <= 0x7fffffffll && rows * columns <= 0x7fffffffll,
             "ll_rotate_by_position: a grid of %lld x %lld", (long long)rows, (long long)columns);
  if (rows > 0) {
    LL_REQUIRE(angles->frame_pairs >= 0 && angles->row_pairs >= 0 && angles->frame_pairs <= p.R / 2 && angles->row_pairs <= p.R / 2 - angles->frame_pairs,
               "ll_rotate_by_position: %d and %d of %d pairs", angles->frame_pairs, angles->row_pairs, p.R / 2);
    p.formed.frame = divisor((uint32_t)(rows * columns));
    p.formed.columns = divisor((uint32_t)columns);
    p.formed.frame_pairs = angles->frame_pairs;
    p.formed.row_pairs = angles->row_pairs;
  }
  p.formed.frequencies = angles->frequencies;
  p.formed.amplitude = angles->amplitude;
  if (tokens == 0 || q->num_heads + k->num_heads == 0) return LL_OK;
  launch_head_norm<true>(p, dtype, tokens, static_cast<hipStream_t>(stream));
  LL_CHECK_LAUNCH("ll_rotate_by_position");
  return LL_OK;
}
