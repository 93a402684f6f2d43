// RMS norm of every head of q and k and the rotation by position, in one pass; and its backward.
//
//   r = 1 / sqrt(mean(x^2) + eps), u = x r w, pairs (a, b) of the first `rot` values turned by the position's angles:
//   y_a = a cos - b sin, y_b = b cos + a sin; the rest of a row is u.
// Backward: g = the turn by minus the angles of dy, h = g w, dx = r (h - x r mean(h x r)), dw = sum over rows of g x r.
//
// Bound by HBM: 4 bytes a value forward (x in, y out), 6 backward (x and dy in, dx out); nothing is kept between the
// two, since r costs no memory once x has to be read again.  A row of d values is d / 16 slots of 16: two vectors of 8
// that hold both halves of 8 pairs (or, with neighbouring pairs, and behind the rotated part, 16 values in a row), so a
// thread turns its own pairs and the only exchange is the row's sum, over 8, 16 or 32 lanes.  The heads of a token share its
// cos and sin: a warp stays with one token and walks its heads.
#include <algorithm>

#include "fm_common.cuh"
#include "fm_kv_cache.cuh"

namespace fm {

struct NormParams {
  const uint16_t* x[2]; uint16_t* y[2];                        // q, k: inputs; outputs (backward: dx)
  const uint16_t* dy[2];
  int64_t xs[2][3], ys[2][3], dys[2][3];                        // strides of batch, token, head
  const void* w[2];                                            // weights, or NULL: ones
  float* part;                                                 // backward: [grid, 2, d] sums of dw
  const float* cos; const float* sin;                          // [table, rot / 2]
  const void* pos; int pos64; int64_t pos_b;                   // [B, S] with that batch stride, or NULL: the token's index
  int B, S, H[2], d, rot, table, w_f32;
  int chunks, per_chunk;                                       // a token's groups of heads are dealt to `chunks` warps
  float eps;
};

// Offsets of the two vectors of 8 of slot `s` in a row.
template <bool INTERLEAVED>
__device__ __forceinline__ void slot_offsets(int s, int rot, int& lo, int& hi) {
  if (INTERLEAVED || s * 16 >= rot) { lo = s * 16; hi = lo + 8; }
  else { lo = s * 8; hi = rot / 2 + lo; }
}

template <bool IS_BF16>
__device__ __forceinline__ void load8(float (&v)[8], const uint16_t* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 f = unpack2<IS_BF16>(w[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
}
template <bool IS_BF16>
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2<IS_BF16>(v[0], v[1]), pack2<IS_BF16>(v[2], v[3]), pack2<IS_BF16>(v[4], v[5]), pack2<IS_BF16>(v[6], v[7]));
}
template <bool IS_BF16>
__device__ __forceinline__ void load_weight8(float (&v)[8], const void* w, int w_f32, int at) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 1.f;
  } else if (w_f32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __ldg(reinterpret_cast<const float*>(w) + at + i);
  } else {
    load8<IS_BF16>(v, reinterpret_cast<const uint16_t*>(w) + at);
  }
}

// Turns the 8 pairs of a slot by the angles (c, s), or by minus them.
template <bool INTERLEAVED, bool BACK>
__device__ __forceinline__ void turn(float (&lo)[8], float (&hi)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float& a = INTERLEAVED ? (i < 4 ? lo[(2 * i) & 7] : hi[(2 * i) & 7]) : lo[i];
    float& b = INTERLEAVED ? (i < 4 ? lo[(2 * i + 1) & 7] : hi[(2 * i + 1) & 7]) : hi[i];
    const float sn = BACK ? -s[i] : s[i], x = a, z = b;
    a = x * c[i] - z * sn;
    b = z * c[i] + x * sn;
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// cos and sin of slot s at the token's position: (1, 0) behind the rotated part, NaN where the table does not have the
// position, so that the mistake shows in the result.
__device__ __forceinline__ void load_angles(const NormParams& p, int64_t b, int t, int s, float (&c)[8], float (&sn)[8]) {
  int64_t pos = t;
  if (p.pos) pos = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[b * p.pos_b + t] : reinterpret_cast<const int32_t*>(p.pos)[b * p.pos_b + t];
  if (s * 16 < p.rot) {
    if (pos >= 0 && pos < p.table) {
      const float4* cp = reinterpret_cast<const float4*>(p.cos + pos * (p.rot / 2) + s * 8);
      const float4* sp = reinterpret_cast<const float4*>(p.sin + pos * (p.rot / 2) + s * 8);
      const float4 c0 = __ldg(cp), c1 = __ldg(cp + 1), s0 = __ldg(sp), s1 = __ldg(sp + 1);
      c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
      sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = sn[i] = __uint_as_float(0x7fffffffu);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) { c[i] = 1.f; sn[i] = 0.f; }
  }
}

// One warp = one token and `per_chunk` of its groups of 32 / LPR heads, q's heads before k's.
template <bool IS_BF16, bool INTERLEAVED, int LPR>
__global__ void __launch_bounds__(256) norm_rotary_fwd_kernel(const NormParams p) {
  const int lane = threadIdx.x & 31, s = lane % LPR, sub = lane / LPR;
  constexpr int HPG = 32 / LPR;
  const int64_t job = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), token = job / p.chunks;
  if (token >= (int64_t)p.B * p.S) return;
  const int64_t b = token / p.S;
  const int t = (int)(token - b * p.S), chunk = (int)(job - token * p.chunks);
  const bool on = s * 16 < p.d;
  int lo, hi;
  slot_offsets<INTERLEAVED>(s, p.rot, lo, hi);
  float c[8], sn[8];
  load_angles(p, b, t, on ? s : p.rot, c, sn);
  const int groups[2] = {(p.H[0] + HPG - 1) / HPG, (p.H[1] + HPG - 1) / HPG};
  const int g0 = chunk * p.per_chunk, g1 = min(g0 + p.per_chunk, groups[0] + groups[1]);
  float wl[8], wh[8];
  int have = -1;
  for (int g = g0; g < g1; ++g) {
    const int which = g >= groups[0], h = (which ? g - groups[0] : g) * HPG + sub;
    if (which != have && on) { load_weight8<IS_BF16>(wl, p.w[which], p.w_f32, lo); load_weight8<IS_BF16>(wh, p.w[which], p.w_f32, hi); }
    have = which;
    const bool live = on && h < p.H[which];
    float a[8] = {}, z[8] = {};
    if (live) {
      const uint16_t* x = p.x[which] + b * p.xs[which][0] + t * p.xs[which][1] + h * p.xs[which][2];
      load8<IS_BF16>(a, x + lo);
      load8<IS_BF16>(z, x + hi);
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + z[i] * z[i];
    const float r = 1.f / sqrtf(row_sum<LPR>(ss) / p.d + p.eps);
    if (!live) continue;
    // (x w is exact where both have 8 bits, and r comes last: three roundings and r's)
#pragma unroll
    for (int i = 0; i < 8; ++i) { a[i] *= wl[i]; z[i] *= wh[i]; }
    turn<INTERLEAVED, false>(a, z, c, sn);
#pragma unroll
    for (int i = 0; i < 8; ++i) { a[i] *= r; z[i] *= r; }
    uint16_t* y = p.y[which] + b * p.ys[which][0] + t * p.ys[which][1] + h * p.ys[which][2];
    store8<IS_BF16>(y + lo, a);
    store8<IS_BF16>(y + hi, z);
  }
}

// Warps walk the (token, chunk) jobs with a stride of the grid and keep the sums of dw of their slots in registers.
template <bool IS_BF16, bool INTERLEAVED, int LPR>
__global__ void __launch_bounds__(256) norm_rotary_bwd_kernel(const NormParams p) {
  extern __shared__ float sums[];                                // [8 warps][2][LPR * 16]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, s = lane % LPR, sub = lane / LPR;
  constexpr int HPG = 32 / LPR;
  const bool on = s * 16 < p.d;
  int lo, hi;
  slot_offsets<INTERLEAVED>(s, p.rot, lo, hi);
  const int groups[2] = {(p.H[0] + HPG - 1) / HPG, (p.H[1] + HPG - 1) / HPG};
  float dw[2][16] = {};
  const int64_t jobs = (int64_t)p.B * p.S * p.chunks;
  for (int64_t job = (int64_t)blockIdx.x * 8 + warp; job < jobs; job += (int64_t)gridDim.x * 8) {
    const int64_t token = job / p.chunks, b = token / p.S;
    const int t = (int)(token - b * p.S), chunk = (int)(job - token * p.chunks);
    float c[8], sn[8];
    load_angles(p, b, t, on ? s : p.rot, c, sn);
    const int g0 = chunk * p.per_chunk, g1 = min(g0 + p.per_chunk, groups[0] + groups[1]);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int from = which ? max(g0 - groups[0], 0) : g0, to = which ? g1 - groups[0] : min(g1, groups[0]);
      if (from >= to) continue;
      float wl[8], wh[8];
      if (on) { load_weight8<IS_BF16>(wl, p.w[which], p.w_f32, lo); load_weight8<IS_BF16>(wh, p.w[which], p.w_f32, hi); }
      for (int g = from; g < to; ++g) {
        const int h = g * HPG + sub;
        const bool live = on && h < p.H[which];
        float a[8] = {}, z[8] = {}, ga[8] = {}, gz[8] = {};
        if (live) {
          const uint16_t* x = p.x[which] + b * p.xs[which][0] + t * p.xs[which][1] + h * p.xs[which][2];
          const uint16_t* dy = p.dy[which] + b * p.dys[which][0] + t * p.dys[which][1] + h * p.dys[which][2];
          load8<IS_BF16>(a, x + lo);
          load8<IS_BF16>(z, x + hi);
          load8<IS_BF16>(ga, dy + lo);
          load8<IS_BF16>(gz, dy + hi);
          turn<INTERLEAVED, true>(ga, gz, c, sn);
        }
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss += a[i] * a[i] + z[i] * z[i];
          dot += live ? ga[i] * wl[i] * a[i] + gz[i] * wh[i] * z[i] : 0.f;
        }
        ss = row_sum<LPR>(ss);
        dot = row_sum<LPR>(dot);
        const float r = 1.f / sqrtf(ss / p.d + p.eps), m = dot * r * r / p.d;
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dw[which][i] += ga[i] * a[i] * r;
          dw[which][8 + i] += gz[i] * z[i] * r;
          a[i] = r * (ga[i] * wl[i] - a[i] * m);
          z[i] = r * (gz[i] * wh[i] - z[i] * m);
        }
        uint16_t* y = p.y[which] + b * p.ys[which][0] + t * p.ys[which][1] + h * p.ys[which][2];
        store8<IS_BF16>(y + lo, a);
        store8<IS_BF16>(y + hi, z);
      }
    }
  }
  if (!p.part) return;
  // sub-rows of the warp, then the warps, in a fixed order
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = dw[which][i];
#pragma unroll
      for (int o = 16; o >= LPR; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (sub == 0 && on) sums[(warp * 2 + which) * LPR * 16 + (i < 8 ? lo + i : hi + i - 8)] = v;
    }
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * p.d; j += 256) {
    const int which = j >= p.d, at = which ? j - p.d : j;
    float v = 0.f;
    for (int k = 0; k < 8; ++k) v += sums[(k * 2 + which) * LPR * 16 + at];
    p.part[(size_t)blockIdx.x * 2 * p.d + j] = v;
  }
}

// dw = sum of the CTAs' sums, in a fixed order: one CTA per 8 columns of the 2 d, 32 threads each.
struct NormSumParams { const float* part; int n, d, w_f32, is_bf16; void* dw[2]; };
__global__ void __launch_bounds__(256) norm_rotary_dw_kernel(const NormSumParams p) {
  grid_dep_wait();
  const int j = blockIdx.x * 8 + (threadIdx.x & 7), k = threadIdx.x >> 3;
  __shared__ float s[32][9];
  float v = 0.f;
  if (j < 2 * p.d)
    for (int i = k; i < p.n; i += 32) v += p.part[(size_t)i * 2 * p.d + j];
  s[k][threadIdx.x & 7] = v;
  __syncthreads();
  if (threadIdx.x >= 8 || j >= 2 * p.d) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) v += s[i][threadIdx.x];
  const int which = j >= p.d, at = which ? j - p.d : j;
  if (!p.dw[which]) return;
  if (p.w_f32) reinterpret_cast<float*>(p.dw[which])[at] = v;
  else if (p.is_bf16) reinterpret_cast<__nv_bfloat16*>(p.dw[which])[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p.dw[which])[at] = __float2half_rn(v);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int sm_count();

// A warp takes all heads of a token where there are tokens enough to fill the chip with warps (cos, sin and the weights
// are loaded once for them), and one group of heads where there are few.
static void norm_plan(const fm_norm_rotary_args* a, NormParams* p) {
  p->B = a->B; p->S = a->S; p->d = a->d;
  const int lpr = a->d <= 128 ? 8 : (a->d <= 256 ? 16 : 32), hpg = 32 / lpr;
  const int groups = (a->Hq + hpg - 1) / hpg + (a->Hk + hpg - 1) / hpg;
  const int64_t tokens = (int64_t)a->B * a->S, warps = (int64_t)sm_count() * 64;
  const int64_t want = tokens > 0 ? (warps + tokens - 1) / tokens : 1;
  p->chunks = (int)std::max<int64_t>(1, std::min<int64_t>(want, groups));
  p->per_chunk = (groups + p->chunks - 1) / p->chunks;
  if (p->per_chunk > 0) p->chunks = (groups + p->per_chunk - 1) / p->per_chunk;
}

static int norm_params(const fm_norm_rotary_args* a, bool back, NormParams* p) {
  FM_REQUIRE(a, FM_ERR_INVALID_ARGUMENT, "norm_rotary: NULL argument");
  FM_REQUIRE(a->dtype == FM_DTYPE_BF16 || a->dtype == FM_DTYPE_FP16, FM_ERR_INVALID_ARGUMENT, "norm_rotary: unknown dtype %d", a->dtype);
  FM_REQUIRE(a->B >= 0 && a->S >= 0 && a->Hq >= 0 && a->Hk >= 0, FM_ERR_INVALID_ARGUMENT, "norm_rotary: negative size");
  FM_REQUIRE(a->d >= 16 && a->d % 16 == 0 && a->d <= 512, FM_ERR_UNSUPPORTED, "norm_rotary: head dim %d is not a multiple of 16 up to 512", a->d);
  FM_REQUIRE(a->rot >= 0 && a->rot <= a->d && a->rot % 16 == 0, FM_ERR_UNSUPPORTED, "norm_rotary: %d rotated values of %d (a multiple of 16)", a->rot, a->d);
  FM_REQUIRE(a->rot == 0 || (a->cos && a->sin && a->table > 0), FM_ERR_INVALID_ARGUMENT, "norm_rotary: cos or sin is NULL");
  FM_REQUIRE(a->positions || a->rot == 0 || a->S <= a->table, FM_ERR_INVALID_ARGUMENT, "norm_rotary: %d tokens, tables of %d positions", a->S, a->table);
  FM_REQUIRE((((uintptr_t)a->cos | (uintptr_t)a->sin) & 15) == 0, FM_ERR_INVALID_ARGUMENT, "norm_rotary: cos or sin is not 16-byte aligned");
  FM_REQUIRE(a->eps >= 0.f, FM_ERR_INVALID_ARGUMENT, "norm_rotary: eps %g", a->eps);
  FM_REQUIRE((int64_t)a->Hq + a->Hk <= 65536, FM_ERR_UNSUPPORTED, "norm_rotary: more than 65536 heads");
  const void* x[2] = {a->q, a->k}; void* y[2] = {a->q_out, a->k_out}; const void* dy[2] = {a->d_q, a->d_k};
  const int64_t* xs[2] = {a->q_stride, a->k_stride}; const int64_t* ys[2] = {a->qo_stride, a->ko_stride};
  const int64_t* ds[2] = {a->dq_stride, a->dk_stride};
  const void* w[2] = {a->q_weight, a->k_weight};
  const int H[2] = {a->Hq, a->Hk};
  for (int i = 0; i < 2; ++i) {
    p->x[i] = (const uint16_t*)x[i]; p->y[i] = (uint16_t*)y[i]; p->dy[i] = back ? (const uint16_t*)dy[i] : nullptr;
    p->w[i] = w[i]; p->H[i] = H[i];
    FM_REQUIRE(((uintptr_t)w[i] & 15) == 0, FM_ERR_INVALID_ARGUMENT, "norm_rotary: a weight is not 16-byte aligned");
    for (int j = 0; j < 3; ++j) {
      p->xs[i][j] = xs[i][j]; p->ys[i][j] = ys[i][j]; p->dys[i][j] = back ? ds[i][j] : 0;
      FM_REQUIRE(p->xs[i][j] % 8 == 0 && p->ys[i][j] % 8 == 0 && p->dys[i][j] % 8 == 0, FM_ERR_INVALID_ARGUMENT,
                 "norm_rotary: strides are not multiples of 8 elements");
    }
    if ((int64_t)a->B * a->S * H[i] == 0) continue;
    FM_REQUIRE(x[i] && y[i] && (!back || dy[i]), FM_ERR_INVALID_ARGUMENT, "norm_rotary: a tensor is NULL");
    FM_REQUIRE((((uintptr_t)x[i] | (uintptr_t)y[i] | (back ? (uintptr_t)dy[i] : 0)) & 15) == 0, FM_ERR_INVALID_ARGUMENT,
               "norm_rotary: a tensor is not 16-byte aligned");
  }
  p->cos = a->cos; p->sin = a->sin; p->pos = a->positions; p->pos64 = a->positions_64; p->pos_b = a->positions_stride;
  p->rot = a->rot; p->table = a->table; p->w_f32 = a->weight_f32;
  p->eps = a->eps;
  p->part = nullptr;
  norm_plan(a, p);
  return FM_OK;
}

static int64_t norm_bwd_grid(const NormParams& p) {
  const int64_t jobs = (int64_t)p.B * p.S * p.chunks, most = (int64_t)sm_count() * 2;
  const int64_t need = (jobs + 7) / 8;
  return need < 1 ? 1 : (need < most ? need : most);
}

template <bool IS_BF16, bool IL>
static int norm_launch(const NormParams& p, bool back, int64_t grid, cudaStream_t s) {
#define FM_NORM(LPR)                                                                                         \
  do {                                                                                                       \
    if (back) norm_rotary_bwd_kernel<IS_BF16, IL, LPR><<<(unsigned)grid, 256, 8 * 2 * LPR * 16 * sizeof(float), s>>>(p); \
    else norm_rotary_fwd_kernel<IS_BF16, IL, LPR><<<(unsigned)grid, 256, 0, s>>>(p);                         \
  } while (0)
  if (p.d <= 128) FM_NORM(8);
  else if (p.d <= 256) FM_NORM(16);
  else FM_NORM(32);
#undef FM_NORM
  count_launches(1);
  FM_CUDA_TRY(cudaGetLastError());
  return FM_OK;
}

static int norm_dispatch(const NormParams& p, const fm_norm_rotary_args* a, bool back, int64_t grid, cudaStream_t s) {
  FM_REQUIRE(grid <= INT_MAX, FM_ERR_UNSUPPORTED, "norm_rotary: too many tokens for one call");
  if (a->dtype == FM_DTYPE_BF16) return a->interleaved ? norm_launch<true, true>(p, back, grid, s) : norm_launch<true, false>(p, back, grid, s);
  return a->interleaved ? norm_launch<false, true>(p, back, grid, s) : norm_launch<false, false>(p, back, grid, s);
}

}  // namespace fm

using namespace fm;

extern "C" FM_API int fm_norm_rotary_fwd(const fm_norm_rotary_args* a, void* stream) {
  NormParams p;
  const int rc = norm_params(a, false, &p);
  if (rc) return rc;
  const int64_t jobs = (int64_t)p.B * p.S * p.chunks;
  if (jobs == 0 || p.per_chunk == 0) return FM_OK;
  return norm_dispatch(p, a, false, (jobs + 7) / 8, (cudaStream_t)stream);
}

extern "C" FM_API size_t fm_norm_rotary_bwd_workspace_bytes(const fm_norm_rotary_args* a) {
  if (!a || a->B < 0 || a->S < 0 || a->Hq < 0 || a->Hk < 0 || a->d < 16 || a->d > 512) return 0;
  NormParams p;
  norm_plan(a, &p);
  return (size_t)norm_bwd_grid(p) * 2 * p.d * sizeof(float);
}

extern "C" FM_API int fm_norm_rotary_bwd(const fm_norm_rotary_args* a, void* stream) {
  NormParams p;
  const int rc = norm_params(a, true, &p);
  if (rc) return rc;
  const bool sums = a->dq_weight || a->dk_weight;
  const int64_t grid = norm_bwd_grid(p);
  if (sums) {
    FM_REQUIRE(a->workspace && a->workspace_bytes >= (size_t)grid * 2 * p.d * sizeof(float) && ((uintptr_t)a->workspace & 15) == 0,
               FM_ERR_WORKSPACE, "fm_norm_rotary_bwd: workspace of %zu bytes", a->workspace_bytes);
    p.part = (float*)a->workspace;
  } else if ((int64_t)p.B * p.S * p.per_chunk == 0) {
    return FM_OK;
  }
  if (const int e = norm_dispatch(p, a, true, grid, (cudaStream_t)stream)) return e;
  if (!sums) return FM_OK;
  const NormSumParams q{p.part, (int)grid, p.d, a->weight_f32, a->dtype == FM_DTYPE_BF16, {a->dq_weight, a->dk_weight}};
  FM_CUDA_TRY(launch_dependent(norm_rotary_dw_kernel, dim3((unsigned)((2 * p.d + 7) / 8)), dim3(256), 0, (cudaStream_t)stream, q));
  count_launches(1);
  return FM_OK;
}
