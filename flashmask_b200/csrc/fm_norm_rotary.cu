// RMS norm of every head of q and k and the rotation by position, in one pass; and its backward.
//
//   r = 1 / sqrt(mean(x^2) + eps), u = x r w, pairs (a, b) of the first `rot` values turned by the position's angles:
//   y_a = a cos - b sin, y_b = b cos + a sin; the rest of a row is u.
// Backward: g = the turn by minus the angles of dy, h = g w, dx = r (h - x r mean(h x r)), dw = sum over rows of g x r.
//
// Bound by HBM: 4 bytes a value forward (x in, y out), 6 backward (x and dy in, dx out); nothing is kept between the
// two, since r costs no memory once x has to be read again.  A row of d values is d / 16 slots of 16: two vectors of 8
// that hold both halves of 8 pairs (or, with neighbouring pairs, and behind the rotated part, 16 values in a row), so a
// thread turns its own pairs and the only exchange is the row's sum, over 4, 8, 16 or 32 lanes.  The heads of a token share its
// cos and sin: a warp stays with one token and walks its heads.
#include <algorithm>

#include "fm_common.cuh"
#include "fm_kv_cache.cuh"

namespace fm {

// n / d for 0 <= n < 2^31 by a product: m = floor(2^(31 + l) / d) + 1 with 2^l >= d is too large by at most d / 2^(31 + l) of 1, which
// times n stays below 1 / d.  A job's place takes two divisions, and many jobs are two groups of rows.
struct Div {
  uint32_t m; int shift;
  void set(int d) {
    int l = 0;
    while ((int64_t)1 << l < d) ++l;
    shift = 31 + l;
    m = d > 0 ? (uint32_t)(((uint64_t)1 << shift) / d + 1) : 0;
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((uint64_t)(uint32_t)n * m >> shift); }
};

struct NormParams {
  const uint16_t* x[2]; uint16_t* y[2];                        // q, k: inputs; outputs (backward: dx)
  const uint16_t* dy[2];
  int64_t xs[2][3], ys[2][3], dys[2][3];                        // strides of batch, token, head
  const void* w[2];                                            // weights, or NULL: ones
  float* part;                                                 // backward: [grid, 2, d] sums of dw
  const float* cos; const float* sin;                          // [table, rot / 2]
  const void* pos; int pos64; int64_t pos_b;                   // [B, S] with that batch stride, or NULL: the token's index
  int B, S, H[2], d, rot, table, w_f32;
  int chunks[2], per_chunk[2];                                 // a token's groups of 32 / LPR heads are dealt to `chunks` jobs
  Div by_S, by_chunks[2];
  float eps, inv_d;
};

// Two fp32 lanes in a 64-bit register (sm_100 packed arithmetic): one instruction for two values.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pair(float a, float b) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpair(f2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ f2 mul(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 fma(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ f2 swap(f2 x) { float a, b; unpair(x, a, b); return pair(b, a); }
__device__ __forceinline__ float sum(f2 x) { float a, b; unpair(x, a, b); return a + b; }

// Offsets of the two vectors of 8 of slot `s` in a row.
template <bool INTERLEAVED>
__device__ __forceinline__ void slot_offsets(int s, int rot, int& lo, int& hi) {
  if (INTERLEAVED || s * 16 >= rot) { lo = s * 16; hi = lo + 8; }
  else { lo = s * 8; hi = rot / 2 + lo; }
}

// A slot: v[0 .. 3] the first vector, v[4 .. 7] the second.
struct Raw { uint4 lo, hi; };
template <bool IS_BF16>
__device__ __forceinline__ void widen(f2 (&v)[8], const Raw& r) {
  const uint32_t w[8] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w, r.hi.x, r.hi.y, r.hi.z, r.hi.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) { const float2 f = unpack2<IS_BF16>(w[i]); v[i] = pair(f.x, f.y); }
}
template <bool IS_BF16>
__device__ __forceinline__ uint32_t narrow(f2 x) { float a, b; unpair(x, a, b); return pack2<IS_BF16>(a, b); }
template <bool IS_BF16>
__device__ __forceinline__ void store(uint16_t* p, int lo, int hi, const f2 (&v)[8]) {
  *reinterpret_cast<uint4*>(p + lo) = make_uint4(narrow<IS_BF16>(v[0]), narrow<IS_BF16>(v[1]), narrow<IS_BF16>(v[2]), narrow<IS_BF16>(v[3]));
  *reinterpret_cast<uint4*>(p + hi) = make_uint4(narrow<IS_BF16>(v[4]), narrow<IS_BF16>(v[5]), narrow<IS_BF16>(v[6]), narrow<IS_BF16>(v[7]));
}
template <bool IS_BF16>
__device__ __forceinline__ void load_weight(f2 (&v)[8], const void* w, int w_f32, int lo, int hi) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = pair(1.f, 1.f);
  } else if (w_f32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __ldg(reinterpret_cast<const float2*>(reinterpret_cast<const float*>(w) + (i < 4 ? lo + 2 * i : hi + 2 * i - 8)));
      v[i] = pair(f.x, f.y);
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(w);
    widen<IS_BF16>(v, Raw{__ldg(reinterpret_cast<const uint4*>(p + lo)), __ldg(reinterpret_cast<const uint4*>(p + hi))});
  }
}

// Turns the 8 pairs of a slot by the angles (c, s), or by minus them.  A register holds two neighbouring angles' values of one
// vector, or, with neighbouring pairs, both values of a pair.
template <bool INTERLEAVED, bool BACK>
__device__ __forceinline__ void turn(f2 (&v)[8], const f2 (&c)[4], const f2 (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float s0, s1;
    unpair(s[i], s0, s1);
    if constexpr (INTERLEAVED) {
      float c0, c1;
      unpair(c[i], c0, c1);
      v[2 * i] = fma(swap(v[2 * i]), BACK ? pair(s0, -s0) : pair(-s0, s0), mul(v[2 * i], pair(c0, c0)));
      v[2 * i + 1] = fma(swap(v[2 * i + 1]), BACK ? pair(s1, -s1) : pair(-s1, s1), mul(v[2 * i + 1], pair(c1, c1)));
    } else {
      const f2 n = pair(-s0, -s1), a = v[i], b = v[4 + i];
      v[i] = fma(b, BACK ? s[i] : n, mul(a, c[i]));
      v[4 + i] = fma(a, BACK ? n : s[i], mul(b, c[i]));
    }
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// cos and sin of slot s at the token's position: (1, 0) behind the rotated part, NaN for the whole row where the table does not
// have the position, so that the mistake shows in the result.  (Without a rotated part positions say nothing.)
__device__ __forceinline__ void load_angles(const NormParams& p, int64_t b, int t, int s, bool on, f2 (&c)[4], f2 (&sn)[4]) {
  int64_t pos = t;
  if (p.pos) pos = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[b * p.pos_b + t] : reinterpret_cast<const int32_t*>(p.pos)[b * p.pos_b + t];
  const bool turned = on && s * 16 < p.rot, there = pos >= 0 && pos < p.table;
  if (turned && there) {
    const ulonglong2* cp = reinterpret_cast<const ulonglong2*>(p.cos + pos * (p.rot / 2) + s * 8);
    const ulonglong2* sp = reinterpret_cast<const ulonglong2*>(p.sin + pos * (p.rot / 2) + s * 8);
    const ulonglong2 c0 = __ldg(cp), c1 = __ldg(cp + 1), s0 = __ldg(sp), s1 = __ldg(sp + 1);
    c[0] = c0.x; c[1] = c0.y; c[2] = c1.x; c[3] = c1.y;
    sn[0] = s0.x; sn[1] = s0.y; sn[2] = s1.x; sn[3] = s1.y;
  } else {
    const bool none = p.rot > 0 && !there;
    const float nan = __uint_as_float(0x7fffffffu);
#pragma unroll
    for (int i = 0; i < 4; ++i) { c[i] = none ? pair(nan, nan) : pair(1.f, 1.f); sn[i] = none ? pair(nan, nan) : pair(0.f, 0.f); }
  }
}

// A warp's job: a token of q or of k and `per_chunk` of its groups of 32 / LPR heads.  All of q's jobs come before k's.
struct NormJob { int64_t b; int t, g0, g1; };
__device__ __forceinline__ NormJob norm_job(const NormParams& p, int which, int job, int groups) {
  const int token = p.by_chunks[which](job), b = p.by_S(token), g0 = (job - token * p.chunks[which]) * p.per_chunk[which];
  return {b, token - b * p.S, g0, min(g0 + p.per_chunk[which], groups)};
}

// Forward.  A warp has one job, and the rows of the next two groups are on their way while one is worked on: 2 x 8192 tokens,
// 32 / 8 heads, d = 128, bf16 (335 MB) in 66 us, 5.1 TB/s, one call behind the other (alone 60: a part of what is written stays in L2); with
// the backward's stream through shared memory alone 70 us.  80 registers: six CTAs of 128 threads to an SM, at 20 to 36 bytes of spills; five
// without any 66 us (4 x 4096 tokens, 16 / 4 heads, d = 64: 26.8 with six, 25.5 with five); at 72 the spills cost more than the seventh brings (64 alone).
template <bool IS_BF16, bool INTERLEAVED, int LPR>
__global__ void __launch_bounds__(128, 6) norm_rotary_fwd_kernel(const __grid_constant__ NormParams p) {
  const int lane = threadIdx.x & 31, s = lane % LPR, sub = lane / LPR;
  constexpr int HPG = 32 / LPR;
  const bool on = s * 16 < p.d;
  int lo, hi;
  slot_offsets<INTERLEAVED>(s, p.rot, lo, hi);
  const int tokens = p.B * p.S, q_jobs = tokens * p.chunks[0];
  int job = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int which = job >= q_jobs;
  if (which) job -= q_jobs;
  if (job >= tokens * p.chunks[which]) return;
  const int H = p.H[which], groups = (H + HPG - 1) / HPG;
  const NormJob j = norm_job(p, which, job, groups);
  const int64_t xh = p.xs[which][2] * HPG, yh = p.ys[which][2] * HPG;
  const uint16_t* x = p.x[which] + j.b * p.xs[which][0] + j.t * p.xs[which][1] + (int64_t)(j.g0 * HPG + sub) * p.xs[which][2];
  uint16_t* y = p.y[which] + j.b * p.ys[which][0] + j.t * p.ys[which][1] + (int64_t)(j.g0 * HPG + sub) * p.ys[which][2];
  auto load = [&](int g) {
    Raw r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (on && g < j.g1 && g * HPG + sub < H) {
      r.lo = __ldcs(reinterpret_cast<const uint4*>(x + lo));
      r.hi = __ldcs(reinterpret_cast<const uint4*>(x + hi));
    }
    x += xh;
    return r;
  };
  Raw next = load(j.g0), after = load(j.g0 + 1);
  f2 c[4], sn[4], w[8];
  load_angles(p, j.b, j.t, s, on, c, sn);
  if (on) load_weight<IS_BF16>(w, p.w[which], p.w_f32, lo, hi);
#pragma unroll 1
  for (int g = j.g0; g < j.g1; ++g) {
    f2 v[8];
    widen<IS_BF16>(v, next);
    next = after;
    after = load(g + 2);
    f2 ss = mul(v[0], v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) ss = fma(v[i], v[i], ss);
    const float r = 1.f / sqrtf(row_sum<LPR>(sum(ss)) * p.inv_d + p.eps);
    // (x w is exact where both have 8 bits, and r comes last: three roundings and r's)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mul(v[i], w[i]);
    turn<INTERLEAVED, false>(v, c, sn);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mul(v[i], pair(r, r));
    if (on && g * HPG + sub < H) store<IS_BF16>(y, lo, hi, v);
    y += yh;
  }
}

// A warp's stream of groups of rows: jobs `first`, `first` + `step`, .. of q or of k, a job being a token and some of its groups of
// HPG = 32 / LPR heads.  Rows of x and dy are copied to shared memory DEPTH groups ahead, across jobs, a row's LPR lanes
// copying its chunks of 16 bytes side by side whatever order they are read in (slots of 32 bytes, a chunk of each at a time, ask L2 for
// every sector twice: neighbouring pairs 140 us instead of 88).  The angles of a job's token go to a ring
// of their own, copied by one row's lanes for all.  (A group read in this step, DEPTH ahead of it, and the angles of the job behind:
// DEPTH + 2 entries where every job is one group.)
// CTAs of 256 threads are resident on an SM as registers (128) and shared memory allow: two, with rows of 32 lanes one, and
// with rows of 16 lanes two at a depth of three (8192 tokens, 16 / 2 heads, d = 256: 50 us; one CTA at a depth of four 66 us).
constexpr int norm_bwd_ctas(int lanes_per_row) { return lanes_per_row == 32 ? 1 : 2; }
template <int LPR>
struct NormStream {
  static constexpr int DEPTH = LPR == 16 ? 3 : 4;
  static constexpr int HPG = 32 / LPR;
  static constexpr int STAGE = 4 * 512, ANGLES = LPR * 64, BYTES = DEPTH * STAGE + (DEPTH + 2) * ANGLES;    // of a warp
  const NormParams& p;
  const int which, lane, s, sub, H, groups;
  const uint32_t ring, angles;
  const int jobs, step;
  // the copies' side
  int job, next_pos, g, g1, stage, entry;
  const uint16_t *x, *dy;

  __device__ __forceinline__ NormStream(const NormParams& p_, int which_, uint32_t smem, int first, int step_)
      : p(p_), which(which_), lane(threadIdx.x & 31), s(lane % LPR), sub(lane / LPR), H(p_.H[which_]),
        groups((p_.H[which_] + HPG - 1) / HPG), ring(smem), angles(smem + DEPTH * STAGE),
        jobs(p_.B * p_.S * p_.chunks[which_]), step(step_), job(first), g(0), g1(0), stage(0), entry(0) {
    next_pos = position(job);
    begin();
  }
  __device__ __forceinline__ NormJob place(int j) const { return norm_job(p, which, j, groups); }
  // the position of job j's token, or -1: not in the tables
  __device__ __forceinline__ int position(int j) const {
    if (j >= jobs) return 0;
    const NormJob a = place(j);
    if (!p.pos) return a.t;
    const int64_t pos = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[a.b * p.pos_b + a.t] : reinterpret_cast<const int32_t*>(p.pos)[a.b * p.pos_b + a.t];
    return pos >= 0 && pos < p.table ? (int)pos : -1;
  }
  // The job's rows from its first group on, and its angles: as load_angles() gives them.
  __device__ __forceinline__ void begin() {
    if (job >= jobs) return;
    const NormJob a = place(job);
    g = a.g0;
    g1 = a.g1;
    const int h = g * HPG + sub;
    x = p.x[which] + a.b * p.xs[which][0] + a.t * p.xs[which][1] + h * p.xs[which][2];
    dy = p.dy[which] + a.b * p.dys[which][0] + a.t * p.dys[which][1] + h * p.dys[which][2];
    const int pos = next_pos;
    next_pos = position(job + step);
    if (sub == 0) {
      const uint32_t to = angles + entry * ANGLES + s * 16;
      const bool turned = s * 16 < p.rot;
      if (turned && pos >= 0) {
        const float *c = p.cos + (int64_t)pos * (p.rot / 2) + s * 8, *n = p.sin + (int64_t)pos * (p.rot / 2) + s * 8;
        cp_async16(to, c, true);
        cp_async16(to + LPR * 16, c + 4, true);
        cp_async16(to + LPR * 32, n, true);
        cp_async16(to + LPR * 48, n + 4, true);
      } else {                                                   // (cos, sin) = (1, 0) behind the rotated part
        const bool none = p.rot > 0 && pos < 0;
        const uint32_t c = none ? 0x7fffffffu : 0x3f800000u, n = none ? 0x7fffffffu : 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" :: "r"(to + LPR * 16 * i), "r"(i < 2 ? c : n) : "memory");
      }
    }
    entry = entry == DEPTH + 1 ? 0 : entry + 1;
  }
  // Where chunk c of the lane's row is in a stage: the lanes of a row read neighbouring chunks or every second one, and eight
  // that are served together then hit different banks.
  __device__ __forceinline__ uint32_t chunk_at(int c) const { return (c >= LPR ? 512 : 0) + (sub * LPR + ((c ^ (c >> 3 & 1)) & (LPR - 1))) * 16; }
  // The copies of the next group; one commit for every call.
  __device__ __forceinline__ void fetch() {
    if (job < jobs) {
      const bool row = g * HPG + sub < H;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = s + i * LPR;
        const uint32_t to = ring + stage * STAGE + chunk_at(c);
        if (row && c * 8 < p.d) {                                  // (what is not copied nobody uses)
          cp_async16(to, x + c * 8, true);
          cp_async16(to + 1024, dy + c * 8, true);
        }
      }
      x += HPG * p.xs[which][2];
      dy += HPG * p.dys[which][2];
      if (++g == g1) { job += step; begin(); }
    }
    stage = stage + 1 == DEPTH ? 0 : stage + 1;
    cp_async_commit();
  }
};

__device__ __forceinline__ uint4 lds_vec(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
template <int LPR>
__device__ __forceinline__ void read_angles(f2 (&c)[4], f2 (&sn)[4], uint32_t at) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 a = lds_vec(at + LPR * 16 * i), b = lds_vec(at + LPR * 16 * (2 + i));
    c[2 * i] = pair(__uint_as_float(a.x), __uint_as_float(a.y)); c[2 * i + 1] = pair(__uint_as_float(a.z), __uint_as_float(a.w));
    sn[2 * i] = pair(__uint_as_float(b.x), __uint_as_float(b.y)); sn[2 * i + 1] = pair(__uint_as_float(b.z), __uint_as_float(b.w));
  }
}

// Backward.  Warps walk q's jobs and then k's with a stride of the grid and keep the sums of dw of their slots in registers.
// 2 x 8192 tokens, 32 / 8 heads, d = 128, bf16 (503 MB) in 87 us with the sum of the CTAs' dw, 5.8 TB/s (4 x 4096, 16 / 4 heads, d = 64, 126 MB: 39 us); with
// the next group's rows in registers 110 us.
template <bool IS_BF16, bool INTERLEAVED, int LPR>
__global__ void __launch_bounds__(256, norm_bwd_ctas(LPR)) norm_rotary_bwd_kernel(const __grid_constant__ NormParams p) {
  using Stream = NormStream<LPR>;
  constexpr int HPG = Stream::HPG;
  extern __shared__ __align__(128) unsigned char smem[];         // [8 warps] rings, sums [8][2][LPR * 16]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, s = lane % LPR, sub = lane / LPR;
  const bool on = s * 16 < p.d;
  int lo, hi;
  slot_offsets<INTERLEAVED>(s, p.rot, lo, hi);
  float* sums = reinterpret_cast<float*>(smem + 8 * Stream::BYTES);
  if (p.part) grid_dep_trigger();                                // (the sum over the CTAs follows, and waits for this kernel's end)
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int step = gridDim.x * 8, w0 = blockIdx.x * 8 + warp, first = which ? step - 1 - w0 : w0;      // (who had a job more of q's has one less of k's)
    __syncwarp();
    Stream in(p, which, smem_u32(smem) + warp * Stream::BYTES, first, step);
    const uint32_t at_lo = in.chunk_at(lo >> 3), at_hi = in.chunk_at(hi >> 3);
#pragma unroll 1
    for (int i = 0; i < Stream::DEPTH; ++i) in.fetch();
    f2 w[8], dw[8];
    if (on) load_weight<IS_BF16>(w, p.w[which], p.w_f32, lo, hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[i] = 0;
    int stage = 0, entry = 0;
    const int64_t yh = p.ys[which][2] * HPG;
#pragma unroll 1
    for (int job = first; job < in.jobs; job += step) {
      const NormJob a = in.place(job);
      uint16_t* y = p.y[which] + a.b * p.ys[which][0] + a.t * p.ys[which][1] + (int64_t)(a.g0 * HPG + sub) * p.ys[which][2];
#pragma unroll 1
      for (int g = a.g0; g < a.g1; ++g) {
        cp_async_wait<Stream::DEPTH - 1>();
        __syncwarp();                                            // (other lanes' copies)
        const uint32_t from = in.ring + stage * Stream::STAGE;
        stage = stage + 1 == Stream::DEPTH ? 0 : stage + 1;
        f2 v[8], d[8], c[4], sn[4];
        widen<IS_BF16>(v, Raw{lds_vec(from + at_lo), lds_vec(from + at_hi)});
        widen<IS_BF16>(d, Raw{lds_vec(from + 1024 + at_lo), lds_vec(from + 1024 + at_hi)});
        read_angles<LPR>(c, sn, in.angles + entry * Stream::ANGLES + s * 16);
        __syncwarp();                                            // every lane has read the stage that is filled now
        in.fetch();
        const bool live = on && g * HPG + sub < in.H;
        turn<INTERLEAVED, true>(d, c, sn);
        f2 ss = mul(v[0], v[0]), dot = mul(mul(d[0], w[0]), v[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) { ss = fma(v[i], v[i], ss); dot = fma(mul(d[i], w[i]), v[i], dot); }
        const float r = 1.f / sqrtf(row_sum<LPR>(live ? sum(ss) : 0.f) * p.inv_d + p.eps), m = row_sum<LPR>(live ? sum(dot) : 0.f) * r * p.inv_d;
        if (live) {
          const float n = -r * r * m;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            d[i] = mul(d[i], pair(r, r));
            dw[i] = fma(d[i], v[i], dw[i]);
            v[i] = fma(v[i], pair(n, n), mul(d[i], w[i]));
          }
          store<IS_BF16>(y, lo, hi, v);
        }
        y += yh;
      }
      entry = entry == Stream::DEPTH + 1 ? 0 : entry + 1;
    }
    cp_async_wait<0>();
    // the warp's rows side by side; the warps below, in a fixed order
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a[2];
      unpair(dw[i], a[0], a[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 16; o >= LPR; o >>= 1) a[e] += __shfl_xor_sync(0xffffffffu, a[e], o);
        if (sub == 0 && on) sums[(warp * 2 + which) * LPR * 16 + (i < 4 ? lo + 2 * i : hi + 2 * i - 8) + e] = a[e];
      }
    }
  }
  if (!p.part) return;
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * p.d; j += 256) {
    const int which = j >= p.d, at = which ? j - p.d : j;
    float v = 0.f;
#pragma unroll
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
    for (int i = k; i < p.n; i += 32 * 5) {                 // (five loads in flight: 296 CTAs' sums are two rounds)
      float x[5];
#pragma unroll
      for (int a = 0; a < 5; ++a) x[a] = i + 32 * a < p.n ? __ldcg(p.part + (size_t)(i + 32 * a) * 2 * p.d + j) : 0.f;
#pragma unroll
      for (int a = 0; a < 5; ++a) v += x[a];
    }
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

static int norm_lanes(int d) { return d <= 64 ? 4 : (d <= 128 ? 8 : (d <= 256 ? 16 : 32)); }       // of a row: LPR

// A warp takes all heads of a token where there are tokens enough to give each of an SM's 24 resident warps one (cos, sin
// and the weights are loaded once for them), and fewer where there are few.  6002 tokens, 16 / 4 heads, d = 96, forward: all heads
// 15.3 us, two halves 18.8 us.  The backward has fewer warps, which walk the jobs; finer jobs, that would even out 3.5 tokens a warp,
// bring nothing (8192 tokens, 32 / 8 heads, d = 128: 51 us either way).
static void norm_plan(const fm_norm_rotary_args* a, NormParams* p) {
  p->B = a->B; p->S = a->S; p->d = a->d;
  const int hpg = 32 / norm_lanes(a->d);
  const int64_t tokens = (int64_t)a->B * a->S, warps = (int64_t)sm_count() * 24;
  const int64_t want = tokens > 0 ? (warps + tokens - 1) / tokens : 1;
  for (int i = 0; i < 2; ++i) {
    const int groups = ((i ? a->Hk : a->Hq) + hpg - 1) / hpg;
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>(want, groups));
    p->per_chunk[i] = (int)std::max<int64_t>(1, (groups + chunks - 1) / chunks);
    p->chunks[i] = (groups + p->per_chunk[i] - 1) / p->per_chunk[i];
    p->by_chunks[i].set(p->chunks[i]);
  }
  p->by_S.set(a->S);
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
  p->inv_d = 1.f / (float)(a->d > 0 ? a->d : 1);
  p->part = nullptr;
  norm_plan(a, p);
  FM_REQUIRE((int64_t)a->B * a->S * std::max(p->chunks[0], p->chunks[1]) < INT_MAX / 2, FM_ERR_UNSUPPORTED, "norm_rotary: too many tokens for one call");
  return FM_OK;
}

static int64_t norm_bwd_grid(const NormParams& p) {
  const int64_t jobs = (int64_t)p.B * p.S * std::max(p.chunks[0], p.chunks[1]), most = (int64_t)sm_count() * norm_bwd_ctas(norm_lanes(p.d));
  return std::max<int64_t>(1, std::min((jobs + 7) / 8, most));
}

template <bool IS_BF16, bool IL, int LPR>
static int norm_launch(const NormParams& p, bool back, cudaStream_t s) {
  if (back) {
    auto kern = norm_rotary_bwd_kernel<IS_BF16, IL, LPR>;
    constexpr int smem = 8 * NormStream<LPR>::BYTES + 8 * 2 * LPR * 16 * 4;
    static std::atomic<uint64_t> done{0};
    FM_CUDA_TRY(allow_smem(kern, smem, done));
    kern<<<(unsigned)norm_bwd_grid(p), 256, smem, s>>>(p);
  } else {
    const int64_t jobs = (int64_t)p.B * p.S * ((int64_t)p.chunks[0] + p.chunks[1]);
    norm_rotary_fwd_kernel<IS_BF16, IL, LPR><<<(unsigned)((jobs + 3) / 4), 128, 0, s>>>(p);
  }
  count_launches(1);
  FM_CUDA_TRY(cudaGetLastError());
  return FM_OK;
}

static int norm_dispatch(const NormParams& p, const fm_norm_rotary_args* a, bool back, cudaStream_t s) {
  const int lpr = norm_lanes(p.d);
#define FM_NORM(BF, IL) (lpr == 4 ? norm_launch<BF, IL, 4>(p, back, s) : lpr == 8 ? norm_launch<BF, IL, 8>(p, back, s) : lpr == 16 ? norm_launch<BF, IL, 16>(p, back, s) : norm_launch<BF, IL, 32>(p, back, s))
  if (a->dtype == FM_DTYPE_BF16) return a->interleaved ? FM_NORM(true, true) : FM_NORM(true, false);
  return a->interleaved ? FM_NORM(false, true) : FM_NORM(false, false);
#undef FM_NORM
}

}  // namespace fm

using namespace fm;

extern "C" FM_API int fm_norm_rotary_fwd(const fm_norm_rotary_args* a, void* stream) {
  NormParams p;
  const int rc = norm_params(a, false, &p);
  if (rc) return rc;
  const int64_t jobs = (int64_t)p.B * p.S * ((int64_t)p.chunks[0] + p.chunks[1]);
  if (jobs == 0) return FM_OK;
  return norm_dispatch(p, a, false, (cudaStream_t)stream);
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
  } else if ((int64_t)p.B * p.S * ((int64_t)p.chunks[0] + p.chunks[1]) == 0) {
    return FM_OK;
  }
  if (const int e = norm_dispatch(p, a, true, (cudaStream_t)stream)) return e;
  if (!sums) return FM_OK;
  const NormSumParams q{p.part, (int)grid, p.d, a->weight_f32, a->dtype == FM_DTYPE_BF16, {a->dq_weight, a->dk_weight}};
  FM_CUDA_TRY(launch_dependent(norm_rotary_dw_kernel, dim3((unsigned)((2 * p.d + 7) / 8)), dim3(256), 0, (cudaStream_t)stream, q));
  count_launches(1);
  return FM_OK;
}
