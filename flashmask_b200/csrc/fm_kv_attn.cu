// Attention of a few query rows per sequence over the 8-bit paged cache.
//
// All query rows of a kv head (queries x heads of its group) read the same keys, so they form one item's rows, eight to
// a column tile of mma.m16n8k16: S^T = K Q^T with the keys as rows and O^T = V^T P^T with the values' dims as rows,
// which fills the instruction from one row on (rows as M would fill a half or a quarter of it).  The payload goes from
// HBM to registers in the order in which the fragments want it and is widened there: fp16 holds every payload value.
//   K: lane (g, t) loads 16-byte chunks t, t + 4, .. of keys g and g + 8; four values of a chunk are one k-step's share
//      of the lane, and Q is laid out with the same permutation of the head dim.
//   V: lane (g, t) loads chunk g of keys 2t, 2t + 1, 2t + 8, 2t + 9; byte pairs of two keys are the A operand's pairs
//      along the keys, and byte 2j, 2j + 1 of chunk g are rows g, g + 8 of O^T's tile j.
//   P^T: the S^T fragment, rounded to fp16 and transposed in registers (movmatrix).
// q in bf16 is brought to fp16 by a power of two per row; p is in (0, 2^8], where fp16 has three bits more than bf16.
//
// Scales.  A page's k scale multiplies the scores.  Its v scale joins the exponent: with x = s + log2(vs) the kernel
// keeps m = max x and p' = 2^(x - m), so that p' V8 sums are in units of 2^m for every page, and the denominator takes
// p' / vs.  Powers of two: both are exact.
//
// Work.  The units (8 warps x 16 keys) of all items are laid out end to end and dealt evenly to one wave of CTAs, each
// a contiguous range: sequences of any lengths load the chip evenly, and nothing about the lengths is needed on the
// host.  A CTA leaves a partial result (fp32 O, l, m) where its range cuts an item; kv_attn_merge_kernel joins them.
// Bound by HBM: (d + dv) bytes a key.
#include <algorithm>

#include "fm_kv_cache.cuh"

namespace fm {

struct KvAttnParams {
  KvGeom g;
  const uint8_t* k; const uint8_t* v; const float* ks; const float* vs;
  const int32_t* table; const int32_t* seqlens; const int32_t* lengths;
  const uint16_t* q; uint16_t* o; float* lse; const float* sink;
  int64_t qs[3];
  int B, S, Hq, G, d, dv, causal, window, bf16;
  int row_tiles;                 // of ROWS rows, per kv head
  float scale_log2;
  int* pre;                      // workspace: [B + 1] first unit of every sequence
  float* part_o; float* part_ml; // workspace: [2 n_cta][ROWS][DV], [2 n_cta][ROWS][2]
  int n_cta;
};

constexpr int KV_WARPS = 8, KV_UNIT = 16 * KV_WARPS;

// What the rows of a sequence may see: rows i < n stand at p0 + i; keys [lo, hi) are seen by one of them at least.
struct KvRange { int len, n, p0, lo, hi; };
__device__ __forceinline__ KvRange kv_range(const KvAttnParams& p, int b) {
  KvRange r;
  r.len = kv_len(p.g, p.seqlens[b]);
  r.n = p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
  r.p0 = r.len - r.n;
  r.hi = r.n > 0 ? r.len : 0;
  r.lo = p.window > 0 ? min(max((int64_t)r.p0 - p.window + 1, (int64_t)0), (int64_t)r.hi) & ~15 : 0;
  return r;
}
__device__ __forceinline__ int kv_units(const KvRange& r) { return max(1, (r.hi - r.lo + KV_UNIT - 1) / KV_UNIT); }

// Keys [lo, hi) that query row i sees; a row that is none sees nothing.
__device__ __forceinline__ void row_range(const KvAttnParams& p, const KvRange& r, int i, int& lo, int& hi) {
  lo = 0; hi = 0;
  if (i >= r.n) return;
  hi = p.causal ? max(r.p0 + i + 1, 0) : r.len;
  if (p.window > 0) lo = (int)max((int64_t)0, (int64_t)r.p0 + i + 1 - p.window);
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// 0x80 in every byte of w that is an e4m3 NaN (0x7f, 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ uint4 ldg_stream(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// DK = ceil(d / 64), VC = bytes of a lane's chunk of V (dv <= 8 VC), NT = column tiles of 8 rows.
template <int DK, int VC, int NT, bool INT8>
__global__ void __launch_bounds__(KV_WARPS * 32, 1) kv_attn_kernel(const KvAttnParams p) {
  constexpr int MT = VC / 2, ROWS = 8 * NT, DV = 8 * VC, VW = VC / 4;       // row tiles of O^T, words of V per lane and key
  extern __shared__ __align__(16) float smem[];
  float* s_o = smem;                                  // [warps][MT * 4][32]
  float* s_m = s_o + KV_WARPS * MT * 128;             // [warps][ROWS]
  float* s_l = s_m + KV_WARPS * ROWS;                 // [warps][ROWS]
  int* s_pre = reinterpret_cast<int*>(s_l + KV_WARPS * ROWS);               // [B + 1]
  __shared__ int s_scan[KV_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int items = p.g.Hkv * p.row_tiles;            // of one sequence

  // first unit of every sequence
  {
    const int per = (p.B + KV_WARPS * 32 - 1) / (KV_WARPS * 32), b0 = tid * per, b1 = min(b0 + per, p.B);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += kv_units(kv_range(p, b)) * items;
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    int at = x - mine;
    for (int w = 0; w < warp; ++w) at += s_scan[w];
    for (int b = b0; b < b1; ++b) { s_pre[b] = at; at += kv_units(kv_range(p, b)) * items; }
    if (b1 == p.B && b0 < b1) s_pre[p.B] = at;
    __syncthreads();
  }
  const int total = s_pre[p.B];
  if (blockIdx.x == 0)
    for (int b = tid; b <= p.B; b += KV_WARPS * 32) p.pre[b] = s_pre[b];
  const int u_end = (int)((int64_t)total * (blockIdx.x + 1) / p.n_cta);
  int u_at = (int)((int64_t)total * blockIdx.x / p.n_cta);

  while (u_at < u_end) {
    // the item of unit u_at
    int b = 0;
    {
      int hi = p.B;                                   // s_pre[b] <= u_at < s_pre[hi]
      while (hi - b > 1) { const int mid = (b + hi) >> 1; if (s_pre[mid] <= u_at) b = mid; else hi = mid; }
    }
    const KvRange r = kv_range(p, b);
    const int units = kv_units(r), in_seq = u_at - s_pre[b], item = in_seq / units, u0 = in_seq - item * units;
    const int u1 = min(units, u0 + u_end - u_at), h = item / p.row_tiles, row0 = (item - h * p.row_tiles) * ROWS;
    const int key0 = r.lo + u0 * KV_UNIT, key1 = min(r.hi, r.lo + u1 * KV_UNIT);
    const int32_t* trow = p.table + b * p.g.table_stride;

    // Q^T fragments (row g of every tile) and what the lane's columns 2t, 2t + 1 see
    uint32_t qf[NT][DK][4][2];
    float f[NT][2], m[NT][2], l[NT][2];
    int lo[NT][2], hi[NT][2], lo_max = 0, hi_min = INT_MAX;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + nt * 8 + g, i = row / p.G;
      const bool on = i < p.S;
      const uint16_t* src = p.q + b * p.qs[0] + i * p.qs[1] + ((int64_t)h * p.G + row - i * p.G) * p.qs[2];
      uint4 x[DK][2];
#pragma unroll
      for (int c = 0; c < DK; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int at = (t + 4 * c) * 16 + j * 8;
          x[c][j] = make_uint4(0, 0, 0, 0);
          if (on && at < p.d) x[c][j] = __ldg(reinterpret_cast<const uint4*>(src + at));
        }
      float row_scale = 1.f;
      if (p.bf16) {
        // largest exponent of the row; fp16 then holds q 2^-e to 2^-24 of the row's largest value
        uint32_t mx = 0;
#pragma unroll
        for (int c = 0; c < DK; ++c)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            mx = __vmaxu2(mx, x[c][j].x & 0x7f807f80u); mx = __vmaxu2(mx, x[c][j].y & 0x7f807f80u);
            mx = __vmaxu2(mx, x[c][j].z & 0x7f807f80u); mx = __vmaxu2(mx, x[c][j].w & 0x7f807f80u);
          }
        mx = max(mx & 0xffffu, mx >> 16);
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = min(max((int)(mx >> 7), 1), 253);
        row_scale = __uint_as_float((uint32_t)e << 23);
        const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
        for (int c = 0; c < DK; ++c)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&x[c][j]);
#pragma unroll
            for (int q = 0; q < 4; ++q) { const float2 v = unpack2<true>(w[q]); w[q] = pack2<false>(v.x * inv, v.y * inv); }
          }
      }
#pragma unroll
      for (int c = 0; c < DK; ++c) {
        qf[nt][c][0][0] = x[c][0].x; qf[nt][c][0][1] = x[c][0].y; qf[nt][c][1][0] = x[c][0].z; qf[nt][c][1][1] = x[c][0].w;
        qf[nt][c][2][0] = x[c][1].x; qf[nt][c][2][1] = x[c][1].y; qf[nt][c][3][0] = x[c][1].z; qf[nt][c][3][1] = x[c][1].w;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f[nt][j] = __shfl_sync(0xffffffffu, row_scale, (2 * t + j) * 4) * p.scale_log2;
        m[nt][j] = -INFINITY;
        l[nt][j] = 0.f;
        const int rj = row0 + nt * 8 + 2 * t + j, ij = rj / p.G;
        row_range(p, r, ij, lo[nt][j], hi[nt][j]);
        if (ij >= p.S) { lo[nt][j] = 0; hi[nt][j] = INT_MAX; }      // (a column of zeros that nobody reads)
        lo_max = max(lo_max, lo[nt][j]);
        hi_min = min(hi_min, hi[nt][j]);
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      lo_max = max(lo_max, __shfl_xor_sync(0xffffffffu, lo_max, o));
      hi_min = min(hi_min, __shfl_xor_sync(0xffffffffu, hi_min, o));
    }
    float o[NT][MT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nt][j][c] = 0.f;

    // the warp's groups of 16 keys: key0 + 16 warp, then every KV_UNIT; their pages are looked up 32 at a time
    const int n_groups = key1 > key0 + 16 * warp ? (key1 - key0 - 16 * warp + KV_UNIT - 1) / KV_UNIT : 0;
    int my_page = -1;
    float my_ks = 0.f, my_vs = 1.f;
    auto look_up = [&](int first) {
      const int i = first + lane;
      my_page = i < n_groups ? kv_page(p.g, trow, key0 + 16 * warp + i * KV_UNIT) : -1;
      if (my_page >= 0) {
        my_ks = __ldg(p.ks + (size_t)my_page * p.g.Hkv + h);
        my_vs = __ldg(p.vs + (size_t)my_page * p.g.Hkv + h);
      }
    };
    uint4 kr[DK][2];
    uint32_t vr[4][VW];
    float ks = 0.f, vs = 1.f;
    int page = -1;
    auto fetch = [&](int i) {
      if ((i & 31) == 0) look_up(i);
      page = __shfl_sync(0xffffffffu, my_page, i & 31);
      ks = __shfl_sync(0xffffffffu, my_ks, i & 31);
      vs = __shfl_sync(0xffffffffu, my_vs, i & 31);
      if (page < 0) return;
      const int slot = (key0 + 16 * warp + i * KV_UNIT) & ((1 << p.g.page_log2) - 1);
      const size_t at = (((size_t)page * p.g.Hkv + h) << p.g.page_log2) + slot;
      const uint8_t* kp = p.k + (at + g) * p.d + t * 16;
#pragma unroll
      for (int c = 0; c < DK; ++c) {
        const bool on = (t + 4 * c) * 16 < p.d;
        kr[c][0] = on ? ldg_stream(kp + c * 64) : make_uint4(0, 0, 0, 0);
        kr[c][1] = on ? ldg_stream(kp + c * 64 + 8 * p.d) : make_uint4(0, 0, 0, 0);
      }
      const uint8_t* vp = p.v + (at + 2 * t) * p.dv + g * (VC < 16 ? VC : 16);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint8_t* q = vp + ((x & 1) + (x >> 1) * 8) * p.dv;
        if constexpr (VC == 8) {
          uint2 v = make_uint2(0, 0);
          if (g * 8 < p.dv) v = __ldg(reinterpret_cast<const uint2*>(q));
          vr[x][0] = v.x; vr[x][1] = v.y;
        } else {
#pragma unroll
          for (int c = 0; c < VC / 16; ++c) {
            const uint4 v = g * 16 + c * 128 < p.dv ? ldg_stream(q + c * 128) : make_uint4(0, 0, 0, 0);
            vr[x][4 * c] = v.x; vr[x][4 * c + 1] = v.y; vr[x][4 * c + 2] = v.z; vr[x][4 * c + 3] = v.w;
          }
        }
      }
    };
    if (n_groups) fetch(0);
    for (int i = 0; i < n_groups; ++i) {
      // this group's payload out of the way of the next one's
      uint4 kc[DK][2];
      uint32_t vc[4][VW];
#pragma unroll
      for (int c = 0; c < DK; ++c) { kc[c][0] = kr[c][0]; kc[c][1] = kr[c][1]; }
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int c = 0; c < VW; ++c) vc[x][c] = vr[x][c];
      const float ks_now = ks, vs_now = vs;
      const bool no_page = page < 0;
      const int k0 = key0 + 16 * warp + i * KV_UNIT;
      if (i + 1 < n_groups) fetch(i + 1);
      if (no_page) continue;

      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[nt][c] = 0.f;
#pragma unroll
      for (int c = 0; c < DK; ++c) {
        const uint32_t a[4] = {kc[c][0].x, kc[c][0].y, kc[c][0].z, kc[c][0].w}, z[4] = {kc[c][1].x, kc[c][1].y, kc[c][1].z, kc[c][1].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t fr[4];
          from_payload4<INT8>(a[j], fr[0], fr[2]);
          from_payload4<INT8>(z[j], fr[1], fr[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<false>(s[nt], fr, qf[nt][c][j][0], qf[nt][c][j][1]);
        }
      }
      // (a NaN scale: the scores of the keys that are seen carry it)
      const float lv = log2f(vs_now), inv_vs = vs_now > 0.f ? 1.f / vs_now : 1.f;
      const bool cut = k0 < lo_max || k0 + 16 > hi_min;
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float fk = f[nt][j] * ks_now;
          float x = s[nt][j] * fk + lv, y = s[nt][2 + j] * fk + lv;
          if (cut) {
            if (k0 + g < lo[nt][j] || k0 + g >= hi[nt][j]) x = -INFINITY;
            if (k0 + g + 8 < lo[nt][j] || k0 + g + 8 >= hi[nt][j]) y = -INFINITY;
          }
          s[nt][j] = x; s[nt][2 + j] = y;
          grow |= fmaxf(x, y) > m[nt][j] + 8.f;
        }
      // the running maximum lags: it moves where a score is more than 2^8 above it
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float x = fmaxf(s[nt][j], s[nt][2 + j]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            x = fmaxf(x, m[nt][j]);
            const float w = x == -INFINITY ? 1.f : fast_exp2(m[nt][j] - x);
            m[nt][j] = x;
            l[nt][j] *= w;
#pragma unroll
            for (int jj = 0; jj < MT; ++jj) { o[nt][jj][j] *= w; o[nt][jj][2 + j] *= w; }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float mm = m[nt][j] == -INFINITY ? 0.f : m[nt][j];
          e[j] = fast_exp2(s[nt][j] - mm);
          e[2 + j] = fast_exp2(s[nt][2 + j] - mm);
          l[nt][j] += (e[j] + e[2 + j]) * inv_vs;
        }
        pb[nt][0] = movmatrix_trans(pack2<false>(e[0], e[1]));
        pb[nt][1] = movmatrix_trans(pack2<false>(e[2], e[3]));
      }
      if constexpr (!INT8) {
        // A NaN among values that a row does not see (slots behind the sequence hold whatever was there) must stay out of
        // that row, and 0 * NaN would not: where a group that some row sees in part holds one, the NaNs are multiplied
        // apart, as ones, with what every row sees.
        uint32_t found = 0;
        if (cut)
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int c = 0; c < VW; ++c) found |= nan_bytes(vc[x][c]);
        if (__any_sync(0xffffffffu, found != 0)) {
          uint32_t sb[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = s[nt][q] == -INFINITY ? 0.f : 1.f;
            sb[nt][0] = movmatrix_trans(pack2<false>(w[0], w[1]));
            sb[nt][1] = movmatrix_trans(pack2<false>(w[2], w[3]));
          }
#pragma unroll
          for (int c = 0; c < VW; ++c) {
            uint32_t bad[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t n = nan_bytes(vc[x][c]);
              bad[x] = (n >> 7) * 0x38u;                   // 1.0 in e4m3
              vc[x][c] &= ~((n >> 7) * 0xffu);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int sel = half ? 0x7362 : 0x5140;
              uint32_t fr[4];
              from_payload4<INT8>(__byte_perm(bad[0], bad[1], sel), fr[0], fr[1]);
              from_payload4<INT8>(__byte_perm(bad[2], bad[3], sel), fr[2], fr[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float seen[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816<false>(seen, fr, sb[nt][0], sb[nt][1]);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  if (seen[q] > 0.f) o[nt][2 * c + half][q] = __uint_as_float(0x7fffffffu);
              }
            }
          }
        }
      }
#pragma unroll
      for (int c = 0; c < VW; ++c) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int sel = half ? 0x7362 : 0x5140;
          uint32_t fr[4];
          from_payload4<INT8>(__byte_perm(vc[0][c], vc[1][c], sel), fr[0], fr[1]);
          from_payload4<INT8>(__byte_perm(vc[2][c], vc[3][c], sel), fr[2], fr[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<false>(o[nt][2 * c + half], fr, pb[nt][0], pb[nt][1]);
        }
      }
    }

    // join the warps: common maximum, scaled sums in warp order
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
        if (g == 0) {
          s_m[warp * ROWS + nt * 8 + 2 * t + j] = m[nt][j];
          s_l[warp * ROWS + nt * 8 + 2 * t + j] = l[nt][j];
        }
      }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == units;
    const int slot = 2 * blockIdx.x + (u0 > 0 ? 0 : 1);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int col = nt * 8 + 2 * t + j;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < KV_WARPS; ++w) top = fmaxf(top, s_m[w * ROWS + col]);
        const float w = m[nt][j] == -INFINITY ? (l[nt][j] == 0.f ? 0.f : 1.f) : fast_exp2(m[nt][j] - top);    // (l NaN without a maximum: kept)
#pragma unroll
        for (int jj = 0; jj < MT; ++jj) {
          s_o[(warp * MT * 4 + jj * 4 + j) * 32 + lane] = o[nt][jj][j] * w;
          s_o[(warp * MT * 4 + jj * 4 + 2 + j) * 32 + lane] = o[nt][jj][2 + j] * w;
        }
      }
      __syncthreads();
      // thread = 4 neighbouring dims of a row
      for (int x = tid; x < 8 * DV / 4; x += KV_WARPS * 32) {
        const int col = x / (DV / 4), dim = (x - col * (DV / 4)) * 4, row = row0 + nt * 8 + col, i = row / p.G;
        constexpr int CH = VC < 16 ? VC : 16;              // bytes of one chunk
        const int chunk = dim / (8 * CH), in = dim - chunk * 8 * CH, gg = in / CH, byte = in - gg * CH + chunk * CH;
        float v[4] = {0.f, 0.f, 0.f, 0.f}, top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < KV_WARPS; ++w) {
          top = fmaxf(top, s_m[w * ROWS + nt * 8 + col]);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            v[c] += s_o[(w * MT * 4 + ((byte + c) >> 1) * 4 + ((byte + c) & 1) * 2 + (col & 1)) * 32 + gg * 4 + (col >> 1)];
        }
#pragma unroll
        for (int w = 0; w < KV_WARPS; ++w) {
          const float mw = s_m[w * ROWS + nt * 8 + col], lw = s_l[w * ROWS + nt * 8 + col];
          sum += mw == -INFINITY ? lw : lw * fast_exp2(mw - top);
        }
        if (i >= p.S) continue;
        if (whole) {
          const int hq = h * p.G + row - i * p.G;
          const float sk = p.sink ? p.sink[hq] * kLog2e : -INFINITY;
          if (p.sink) {
            const float up = fmaxf(top, sk), w = top == -INFINITY ? 1.f : fast_exp2(top - up);
            sum = sum * w + (sk == -INFINITY ? 0.f : fast_exp2(sk - up));
            v[0] *= w; v[1] *= w; v[2] *= w; v[3] *= w;
            top = up;
          }
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          if (dim == 0) p.lse[((int64_t)b * p.Hq + hq) * p.S + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
          if (dim < p.dv) {
            const uint2 w = p.bf16 ? make_uint2(pack2<true>(v[0] * inv, v[1] * inv), pack2<true>(v[2] * inv, v[3] * inv))
                                   : make_uint2(pack2<false>(v[0] * inv, v[1] * inv), pack2<false>(v[2] * inv, v[3] * inv));
            *reinterpret_cast<uint2*>(p.o + (((int64_t)b * p.S + i) * p.Hq + hq) * p.dv + dim) = w;
          }
        } else {
          *reinterpret_cast<float4*>(p.part_o + ((size_t)slot * ROWS + nt * 8 + col) * DV + dim) = make_float4(v[0], v[1], v[2], v[3]);
          if (dim == 0) *reinterpret_cast<float2*>(p.part_ml + ((size_t)slot * ROWS + nt * 8 + col) * 2) = make_float2(top, sum);
        }
      }
      __syncthreads();
    }
    u_at += u1 - u0;
  }
  grid_dep_trigger();
}

// One CTA = one query row (of a kv head's rows) of one item that was cut: its parts lie in consecutive CTAs' slots.
// Four groups of 32 lanes take the parts in turn and are then joined in order.
template <int DV, int ROWS>
__global__ void __launch_bounds__(128) kv_attn_merge_kernel(const KvAttnParams p) {
  constexpr int PER = DV / 32;
  __shared__ float s_v[4][DV], s_m[4], s_l[4];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, b = blockIdx.z, h = blockIdx.y, row = blockIdx.x;
  grid_dep_wait();
  const int64_t total = p.pre[p.B], n = p.n_cta;
  const int first = p.pre[b], units = (p.pre[b + 1] - first) / (p.g.Hkv * p.row_tiles), tile = row / ROWS;
  const int64_t s0 = first + (int64_t)(h * p.row_tiles + tile) * units, s1 = s0 + units - 1;
  const int c0 = (int)(((s0 + 1) * n - 1) / total), c1 = (int)(((s1 + 1) * n - 1) / total);
  if (c0 == c1) return;                                   // done by one CTA
  float m = -INFINITY, l = 0.f, v[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) v[x] = 0.f;
  for (int c = c0 + grp; c <= c1; c += 4) {
    const size_t at = (size_t)(2 * c + (c == c0 ? 1 : 0)) * ROWS + row - tile * ROWS;
    // (no unit of the item in this CTA: an empty range, as with fewer units than CTAs)
    if (total * (c + 1) / n == total * c / n) continue;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
    float y[PER];
    if constexpr (PER == 2) { const float2 q = *reinterpret_cast<const float2*>(p.part_o + at * DV + lane * 2); y[0] = q.x; y[1] = q.y; }
    else
#pragma unroll
      for (int x = 0; x < PER; x += 4) {
        const float4 q = *reinterpret_cast<const float4*>(p.part_o + at * DV + lane * PER + x);
        y[x] = q.x; y[x + 1] = q.y; y[x + 2] = q.z; y[x + 3] = q.w;
      }
    const float top = fmaxf(m, ml.x), w0 = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : fast_exp2(m - top),
                w1 = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - top);
    l = l * w0 + ml.y * w1;
    m = top;
#pragma unroll
    for (int x = 0; x < PER; ++x) v[x] = v[x] * w0 + y[x] * w1;
  }
#pragma unroll
  for (int x = 0; x < PER; ++x) s_v[grp][lane * PER + x] = v[x];
  if (lane == 0) { s_m[grp] = m; s_l[grp] = l; }
  __syncthreads();
  const int i = row / p.G, hq = h * p.G + row - i * p.G;
  const float sk = p.sink ? p.sink[hq] * kLog2e : -INFINITY;
  float top = sk;
#pragma unroll
  for (int q = 0; q < 4; ++q) top = fmaxf(top, s_m[q]);
  float w[4], sum = sk == -INFINITY ? 0.f : fast_exp2(sk - top);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    w[q] = s_m[q] == -INFINITY ? (s_l[q] == 0.f ? 0.f : 1.f) : fast_exp2(s_m[q] - top);
    sum += s_l[q] * w[q];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (threadIdx.x == 0) p.lse[((int64_t)b * p.Hq + hq) * p.S + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  for (int dim = threadIdx.x; dim < p.dv; dim += 128) {
    float x = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) x += s_v[q][dim] * w[q];
    x *= inv;
    const size_t at = (((int64_t)b * p.S + i) * p.Hq + hq) * p.dv + dim;
    if (p.bf16) reinterpret_cast<__nv_bfloat16*>(p.o)[at] = __float2bfloat16_rn(x);
    else reinterpret_cast<__half*>(p.o)[at] = __float2half_rn(x);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int sm_count();
int kv_geometry(const fm_kv_cache* c, const fm_kv_args* a, KvGeom* g);

constexpr int KV_MAX_B = 8192;                      // first units of the sequences are kept in shared memory

struct KvAttnPlan { int vc, nt, n_cta; size_t pre_bytes, bytes; };
static KvAttnPlan kv_attn_plan(const fm_kv_cache* c, const fm_kv_args* a) {
  KvAttnPlan pl;
  const int rows = a->S * (a->Hq / c->Hkv);
  pl.vc = c->dv <= 64 && c->d <= 64 ? 8 : (c->dv <= 128 ? 16 : 32);
  pl.nt = rows <= 8 || pl.vc == 32 ? 1 : 2;
  pl.n_cta = sm_count();
  pl.pre_bytes = ((size_t)(a->B + 1) * sizeof(int) + 15) & ~(size_t)15;
  pl.bytes = pl.pre_bytes + (size_t)2 * pl.n_cta * pl.nt * 8 * (8 * pl.vc + 2) * sizeof(float);
  return pl;
}

template <int DK, int VC, int NT, bool INT8>
static int launch_kv_attn(const KvAttnParams& p, cudaStream_t s) {
  auto kern = kv_attn_kernel<DK, VC, NT, INT8>;
  const size_t smem = (size_t)(KV_WARPS * (VC / 2) * 128 + 2 * KV_WARPS * 8 * NT + p.B + 1) * 4;
  FM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
  kern<<<p.n_cta, KV_WARPS * 32, smem, s>>>(p);
  count_launches(1);
  FM_CUDA_TRY(cudaGetLastError());
  FM_CUDA_TRY(launch_dependent(kv_attn_merge_kernel<8 * VC, 8 * NT>, dim3(p.S * p.G, p.g.Hkv, p.B), dim3(128), 0, s, p));
  count_launches(1);
  return FM_OK;
}

template <bool INT8>
static int dispatch_kv_attn(const KvAttnParams& p, const KvAttnPlan& pl, cudaStream_t s) {
  if (pl.vc == 32) return launch_kv_attn<4, 32, 1, INT8>(p, s);
  if (p.d == 192) return pl.nt == 1 ? launch_kv_attn<3, 16, 1, INT8>(p, s) : launch_kv_attn<3, 16, 2, INT8>(p, s);
  if (pl.vc == 16) return pl.nt == 1 ? launch_kv_attn<2, 16, 1, INT8>(p, s) : launch_kv_attn<2, 16, 2, INT8>(p, s);
  return pl.nt == 1 ? launch_kv_attn<1, 8, 1, INT8>(p, s) : launch_kv_attn<1, 8, 2, INT8>(p, s);
}

}  // namespace fm

using namespace fm;

static bool kv_attn_sizes(const fm_kv_cache* c, const fm_kv_args* a) {
  return c && a && c->Hkv > 0 && c->d > 0 && c->dv > 0 && a->B >= 0 && a->S >= 0 && a->Hq > 0 && a->Hq % c->Hkv == 0;
}

extern "C" FM_API size_t fm_kv_attention_workspace_bytes(const fm_kv_cache* c, const fm_kv_args* a) {
  return kv_attn_sizes(c, a) ? kv_attn_plan(c, a).bytes : 0;
}

extern "C" FM_API int fm_kv_attention(const fm_kv_cache* c, const fm_kv_args* a, void* stream) {
  KvAttnParams p;
  const int rc = kv_geometry(c, a, &p.g);
  if (rc) return rc;
  FM_REQUIRE(kv_attn_sizes(c, a), FM_ERR_INVALID_ARGUMENT, "fm_kv_attention: Hq=%d is no multiple of Hkv=%d", a->Hq, c->Hkv);
  FM_REQUIRE(a->window >= 0 && (a->causal || a->window == 0), FM_ERR_INVALID_ARGUMENT, "fm_kv_attention: window %d (causal %d)", a->window, a->causal);
  if (a->B == 0 || a->S == 0) return FM_OK;
  FM_REQUIRE(a->q && a->o && a->lse && a->seqlens, FM_ERR_INVALID_ARGUMENT, "fm_kv_attention: q, o, lse or seqlens is NULL");
  FM_REQUIRE((((uintptr_t)a->q | (uintptr_t)a->o) & 15) == 0, FM_ERR_INVALID_ARGUMENT, "fm_kv_attention: q or o is not 16-byte aligned");
  for (int i = 0; i < 3; ++i) {
    FM_REQUIRE(a->q_stride[i] % 8 == 0, FM_ERR_INVALID_ARGUMENT, "fm_kv_attention: strides are not multiples of 8 elements");
    p.qs[i] = a->q_stride[i];
  }
  FM_REQUIRE(a->B <= KV_MAX_B, FM_ERR_UNSUPPORTED, "fm_kv_attention: %d sequences, at most %d", a->B, KV_MAX_B);
  const KvAttnPlan pl = kv_attn_plan(c, a);
  const int64_t G = a->Hq / c->Hkv, rows = a->S * G, tiles = (rows + pl.nt * 8 - 1) / (pl.nt * 8);
  const int64_t units = ((int64_t)a->max_pages * c->page_size + 31) / KV_UNIT + 1;
  FM_REQUIRE(rows < INT_MAX && units * tiles <= (INT_MAX - 1) / c->Hkv / a->B, FM_ERR_UNSUPPORTED, "fm_kv_attention: too many rows and keys for one call");
  FM_REQUIRE(a->workspace && a->workspace_bytes >= pl.bytes && ((uintptr_t)a->workspace & 15) == 0, FM_ERR_WORKSPACE,
             "fm_kv_attention: workspace of %zu bytes, %zu needed", a->workspace_bytes, pl.bytes);
  p.k = (const uint8_t*)c->k; p.v = (const uint8_t*)c->v; p.ks = c->k_scale; p.vs = c->v_scale;
  p.table = a->page_table; p.seqlens = a->seqlens; p.lengths = a->lengths;
  p.q = (const uint16_t*)a->q; p.o = (uint16_t*)a->o; p.lse = a->lse; p.sink = a->sink;
  p.B = a->B; p.S = a->S; p.Hq = a->Hq; p.G = (int)G; p.d = c->d; p.dv = c->dv;
  p.causal = a->causal; p.window = a->window; p.bf16 = a->dtype == FM_DTYPE_BF16;
  p.row_tiles = (int)tiles;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.n_cta = pl.n_cta;
  p.pre = (int*)a->workspace;
  p.part_o = (float*)((char*)a->workspace + pl.pre_bytes);
  p.part_ml = p.part_o + (size_t)2 * pl.n_cta * pl.nt * 8 * 8 * pl.vc;
  return c->dtype == FM_CACHE_INT8 ? dispatch_kv_attn<true>(p, pl, (cudaStream_t)stream) : dispatch_kv_attn<false>(p, pl, (cudaStream_t)stream);
}
