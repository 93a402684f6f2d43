// Attention of a few query rows per sequence over the 8-bit paged cache.
//
// All query rows of a kv head (queries x heads of its group) read the same keys, so they form one item's rows, eight to
// a column tile of mma.m16n8k16: S^T = K Q^T with the keys as rows and O^T = V^T P^T with the values' dims as rows,
// which fills the instruction from one row on (rows as M would fill a half or a quarter of it).  The payload is copied to a
// ring in shared memory by its bytes, and a lane reads it in the order in which the fragments want it and widens it in
// registers: fp16 holds every payload value.
//   K: lane (g, t) reads 16-byte chunks t, t + 4, .. of keys g and g + 8; four values of a chunk are one k-step's share
//      of the lane, and Q is laid out with the same permutation of the head dim.
//   V: lane (g, t) reads chunk g of keys 2t, 2t + 1, 2t + 8, 2t + 9; byte pairs of two keys are the A operand's pairs
//      along the keys, and byte 2j, 2j + 1 of chunk g are rows g, g + 8 of O^T's tile j.
//   P^T: the S^T fragment, rounded to fp16 and transposed in registers (movmatrix).
// q in bf16 is brought to fp16 by a power of two per row; p is in (0, 2^15], where fp16 has three bits more than bf16.
//
// Scales.  A page's k scale multiplies the scores.  Its v scale joins the exponent: with x = s + log2(vs) and m at the
// largest x the kernel keeps p' = 2^(x - m), so that sums of p' V8 are in units of 2^m for every page, and the
// denominator takes p' / vs.  Powers of two: both are exact.
//
// Work.  The units (4 warps x 32 keys) of all items are laid out end to end and dealt evenly to one wave of CTAs, each
// a contiguous range: sequences of any lengths load the chip evenly, and nothing about the lengths is needed on the
// host.  A warp's copies run on across items.  A CTA leaves a partial result (fp32 O, l, m) where its range cuts an item;
// kv_attn_merge_kernel joins them.
//
// Bound by HBM, (d + dv) bytes a key, once a call is long: 8 x 32768 keys, 32 / 8 heads, d = 128, one token: 88 us, 6.1
// TB/s; 8 x 8192: 30 us, 4.5 TB/s (of which 4 us until the first data are there, 4 us behind the last, and CTAs that end between 20 and
// 26 us: memory serves them unevenly); 64 x 4096, d = 64, int8: 55 us, 4.9 TB/s.  From 16 rows on the dependent instructions of too few
// warps bind, 8 x 8192 with 16 rows 36 us and 32 rows 51 us: 255 registers (with 32 rows, d = 128, e4m3 136 bytes of spills besides) leave two CTAs to an SM.
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
  float* part_o; float* part_ml; // workspace: [2 n_cta][ROWS][DV], [2 n_cta][ROWS][2]
  int n_cta;
};

// A warp works on blocks of 32 keys (two groups of 16), the four blocks of a unit side by side.
constexpr int KV_WARPS = 4, KV_BLOCK = 32, KV_UNIT = KV_BLOCK * KV_WARPS, KV_INFO = 64;

// DK = ceil(d / 64), VC = bytes of a lane's chunk of V (dv <= 8 VC), NT = column tiles of 8 rows.
// Several CTAs share an SM: while one waits or joins its warps the others' copies and products go on.
template <int DK, int VC, int NT>
struct KvCfg {
  static constexpr int KP = DK * 64, VP = VC * 8;                // bytes of a key's and a value's row in shared memory
  static constexpr int GROUP = 16 * (KP + VP), STAGE = 2 * GROUP;          // a group and a block of a warp
  static constexpr int CTAS = VC > 16 ? 1 : (DK > 2 ? 2 : (DK == 1 ? (NT == 1 ? 4 : (NT == 2 ? 3 : 2)) : (NT == 1 ? 3 : 2)));    // by their registers
  static constexpr int STAGES = (CTAS == 1 ? 192 : (CTAS == 2 ? (NT > 2 ? 80 : 96) : (CTAS == 3 ? 64 : 48))) * 1024 / (KV_WARPS * STAGE);
  static constexpr int RING = KV_WARPS * STAGES * STAGE;
  static constexpr int ROWS = 8 * NT, DV = 8 * VC, MT = VC / 2;  // MT row tiles of O^T
  static constexpr int FIT = STAGE / (MT * 512), JOIN = FIT >= NT ? NT : (NT % 2 == 0 && FIT >= 2 ? 2 : 1);    // column tiles of O joined together: a stage holds them
  static constexpr int Q = NT * DK * 4 * 32 * 8;                 // Q^T fragments
  static constexpr int FIXED = RING + Q + KV_WARPS * KV_INFO * 16 + 2 * KV_WARPS * ROWS * 4 + ROWS * 20;   // .., info, m, l, limits, scales, totals
  static_assert(STAGES >= 2 && 2 * STAGES <= KV_INFO - 32, "a block is copied while another is used");
  static_assert(JOIN > 0 && NT % JOIN == 0 && NT <= KV_WARPS, "O fits the stage of the last block; a warp for every tile of queries");
};

// Byte offsets of 16-byte chunk c of row r of a group in shared memory.  The reads of eight lanes that are served
// together go to chunks t .. t + 3 of two neighbouring keys, and to chunks g, g + 1 of values 2t, t = 0 .. 3: the
// permutations put these on different banks.
template <int DK>
__device__ __forceinline__ uint32_t k_at(int r, int c) { return r * (DK * 64) + ((DK & 1 ? c : c ^ ((r & 1) << 2)) << 4); }
template <int VC>
__device__ __forceinline__ uint32_t v_at(int r, int c) { return r * (VC * 8) + ((VC == 8 ? c ^ (r >> 1 & 3) : c ^ ((r >> 1 & 3) << 1)) << 4); }

// What the rows of a sequence may see: rows i < n stand at p0 + i; keys [lo, hi) are seen by one of them at least.
struct KvRange { int len, n, p0, lo, hi; };
__device__ __forceinline__ KvRange kv_range(const KvAttnParams& p, int b) {
  KvRange r;
  r.len = kv_len(p.g, p.seqlens[b]);
  r.n = p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
  r.p0 = r.len - r.n;
  r.hi = r.n > 0 ? r.len : 0;
  r.lo = p.window > 0 ? min(max(r.p0 - p.window + 1, 0), r.hi) & ~(KV_BLOCK - 1) : 0;      // (the host keeps window and S below 2^30)
  return r;
}
__device__ __forceinline__ int kv_units(const KvRange& r) { return max(1, (r.hi - r.lo + KV_UNIT - 1) / KV_UNIT); }

// How the units are dealt.  Every item counts `extra` slots behind its units, for the time that loading its queries and
// joining its sums takes: about a unit's, so that CTAs with many short sequences end when the others do (64 ragged
// sequences, d = 64: CTAs ended between 37 and 58 us without).  None where every unit gets a CTA of its own.  The slots are dealt to n CTAs, the
// first slots % n of which get one more.
struct KvDeal {
  int n, extra, slots;
  __device__ __forceinline__ KvDeal(int n_cta, int units, int n_items) : n(min(n_cta, units)), extra(units > n_cta ? 1 : 0), slots(units + n_items * extra) {}
  __device__ __forceinline__ int first_slot(int c) const { return slots / n * c + min(c, slots % n); }
  __device__ __forceinline__ int cta_of(int slot) const {
    const int q = slots / n, r = slots % n;
    return slot < r * (q + 1) ? slot / (q + 1) : r + (slot - r * (q + 1)) / q;
  }
};

// Keys [lo, hi) that query row i sees; a row that is none sees nothing.
__device__ __forceinline__ void row_range(const KvAttnParams& p, const KvRange& r, int i, int& lo, int& hi) {
  lo = 0; hi = 0;
  if (i >= r.n) return;
  hi = p.causal ? max(r.p0 + i + 1, 0) : r.len;
  if (p.window > 0) lo = max(0, r.p0 + i + 1 - p.window);
}

// (not volatile, as the products: the compiler may order what does not depend on each other)
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// What a range of units of one item is: the item, and which of its keys.
struct KvSegment {
  int b, h, row0, units, u0, u1, key0;
  KvRange r;
  __device__ __forceinline__ KvSegment of_lane(int x) const {
    auto s = [&](int v) { return __shfl_sync(0xffffffffu, v, x); };
    return {s(b), s(h), s(row0), s(units), s(u0), s(u1), s(key0), {s(r.len), s(r.n), s(r.p0), s(r.lo), s(r.hi)}};
  }
};

// FULL: d = 64 DK and dv = 8 VC, known to the compiler.
// The loops over chunks of the head dim and over the two groups stay loops: short calls run every instruction once or
// twice, and wait for instructions more than for anything else.
template <int DK, int VC, int NT, bool INT8, bool FULL>
__global__ void __launch_bounds__(KV_WARPS * 32, KvCfg<DK, VC, NT>::CTAS) kv_attn_kernel(const __grid_constant__ KvAttnParams p) {
  using Cfg = KvCfg<DK, VC, NT>;
  constexpr int MT = Cfg::MT, ROWS = Cfg::ROWS, DV = Cfg::DV, VW = VC / 4, STAGES = Cfg::STAGES, JOIN = Cfg::JOIN;    // VW words of V per lane and key
  extern __shared__ __align__(128) unsigned char smem[];
  uint2* s_q = reinterpret_cast<uint2*>(smem + Cfg::RING);                  // [NT][DK][4][32]
  float4* s_info = reinterpret_cast<float4*>(smem + Cfg::RING + Cfg::Q);    // [warps][KV_INFO]
  float* s_m = reinterpret_cast<float*>(s_info + KV_WARPS * KV_INFO);       // [warps][ROWS]
  float* s_l = s_m + KV_WARPS * ROWS;                 // [warps][ROWS]
  int2* s_lim = reinterpret_cast<int2*>(s_l + KV_WARPS * ROWS);             // [ROWS] keys that a row sees
  float* s_f = reinterpret_cast<float*>(s_lim + ROWS);                      // [ROWS] scale of a row of q
  float2* s_tot = reinterpret_cast<float2*>(s_f + ROWS);                    // [ROWS] maximum and sum of a row
  int* s_pre = reinterpret_cast<int*>(s_tot + ROWS);  // [B + 1] first unit of every sequence
  __shared__ int s_scan[KV_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int d = FULL ? DK * 64 : p.d, dv = FULL ? VC * 8 : p.dv;
  grid_dep_trigger();                                 // (the merge waits for this kernel's end before it reads anything)
  const int items = p.g.Hkv * p.row_tiles;            // of one sequence
  if (p.B <= 32) {
    // (every warp for itself, without a barrier)
    int x = lane < p.B ? kv_units(kv_range(p, lane)) * items : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    s_pre += warp * 33;
    if (lane < p.B) s_pre[lane + 1] = x;
    if (lane == 0) s_pre[0] = 0;
    __syncwarp();
  } else {
    const int per = (p.B + KV_WARPS * 32 - 1) / (KV_WARPS * 32), b0 = tid * per, b1 = min(b0 + per, p.B);
    int mine = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) { s_pre[b] = mine; mine += kv_units(kv_range(p, b)) * items; }
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    int at = x - mine;
    for (int w = 0; w < warp; ++w) at += s_scan[w];
#pragma unroll 1
    for (int b = b0; b < b1; ++b) s_pre[b] += at;
    if (b1 == p.B && b0 < b1) s_pre[p.B] = at + mine;
    __syncthreads();
  }
  const KvDeal deal(p.n_cta, s_pre[p.B], p.B * items);
  if (blockIdx.x >= deal.n) return;
  // units before a slot
  auto units_before = [&](int slot) {
    if (deal.extra == 0 || slot >= deal.slots) return min(slot, s_pre[p.B]);
    int b = 0, hi = p.B;
#pragma unroll 1
    while (hi - b > 1) { const int mid = (b + hi) >> 1; if (s_pre[mid] + mid * items <= slot) b = mid; else hi = mid; }
    const int units = (s_pre[b + 1] - s_pre[b]) / items, in_seq = slot - s_pre[b] - b * items, item = in_seq / (units + 1);
    return s_pre[b] + item * units + min(in_seq - item * (units + 1), units);
  };
  const int edge = units_before(deal.first_slot(blockIdx.x + (lane & 1)));          // (both ends of the range at once)
  const int u_begin = __shfl_sync(0xffffffffu, edge, 0), n_units = __shfl_sync(0xffffffffu, edge, 1) - u_begin;
  if (n_units == 0) return;

  // The part of the item of unit u that this CTA has from u on.
  auto segment = [&](int u) {
    KvSegment s;
    int b = 0, hi = p.B;                              // s_pre[b] <= u < s_pre[hi]
#pragma unroll 1
    while (hi - b > 1) { const int mid = (b + hi) >> 1; if (s_pre[mid] <= u) b = mid; else hi = mid; }
    s.b = b;
    s.r = kv_range(p, b);
    s.units = kv_units(s.r);
    const int in_seq = u - s_pre[b], item = in_seq / s.units;
    s.u0 = in_seq - item * s.units;
    s.u1 = min(s.units, s.u0 + u_begin + n_units - u);
    s.h = p.row_tiles == 1 ? item : item / p.row_tiles;
    s.row0 = (item - s.h * p.row_tiles) * ROWS;
    s.key0 = s.r.lo + s.u0 * KV_UNIT;
    return s;
  };

  // Groups j = 2 i + (0, 1) of the warp's block in unit u_begin + i.  They are looked up 32 at a time, a lane each and across
  // items, and kept in shared memory: the index of the group in the cache (-1: none), which the copies need, and (ks,
  // log2 vs, 1 / vs) behind the first copies.  A group that is none has scores of -inf and values of 0.  In steps, between which
  // the first round has other work to do: the page number is asked for, the place stored, the scales asked for, and stored.
  float4* info = s_info + warp * KV_INFO;
  KvSegment ahead = {};
  int number = -1, page = -1, key = 0;
  float ks = 0.f, vs = 1.f;
  auto ask_page = [&](int first) {
    const int i = (first + lane) >> 1;
    number = -1;
    if (i < n_units) {
      ahead = segment(u_begin + i);
      key = ahead.key0 + KV_BLOCK * warp + (lane & 1) * 16;
      if (key < ahead.r.hi) number = kv_page_number(p.g, p.table + ahead.b * p.g.table_stride, key);
    }
  };
  auto store_place = [&](int first) {
    page = kv_page_in(p.g, number);
    const int at = page < 0 ? -1 : ((page * p.g.Hkv + ahead.h) << (p.g.page_log2 - 4)) + ((key & ((1 << p.g.page_log2) - 1)) >> 4);
    info[(first + lane) & (KV_INFO - 1)].w = __int_as_float(at);
    __syncwarp();
  };
  auto ask_scale = [&]() {
    ks = 0.f; vs = 1.f;
    if (page >= 0) {
      const int64_t ph = (int64_t)page * p.g.Hkv + ahead.h;
      ks = __ldg(p.ks + ph);
      vs = __ldg(p.vs + ph);
    }
  };
  auto store_scale = [&](int first) {
    float4* to = &info[(first + lane) & (KV_INFO - 1)];
    to->x = ks;
    to->y = page >= 0 ? log2f(vs) : -INFINITY;
    to->z = vs > 0.f ? 1.f / vs : 1.f;                     // (not needed of a NaN scale: the scores of the keys that are seen are NaN)
    __syncwarp();
  };
  const uint32_t ring = smem_u32(smem) + warp * STAGES * Cfg::STAGE;
  // The copies of the warp's block in unit i, 16 bytes a lane; zeros behind the head dim.  One commit for every call.
  auto fetch = [&](int i, int stage) {
    if (i < n_units) {
      if ((i & 15) == 0) {
        if (i > 0) ask_page(2 * i);
        store_place(2 * i);
      }
#pragma unroll 1
      for (int hh = 0; hh < 2; ++hh) {
        const int at = __float_as_int(info[(2 * i + hh) & (KV_INFO - 1)].w);
        const uint32_t to = ring + stage * Cfg::STAGE + hh * Cfg::GROUP;
        const uint8_t *kp = p.k + (int64_t)max(at, 0) * 16 * d, *vp = p.v + (int64_t)max(at, 0) * 16 * dv;
#pragma unroll
        for (int x = 0; x < 2 * DK; ++x) {
          const int q = lane + 32 * x, r = q / (4 * DK), c = q - r * 4 * DK;
          const bool on = at >= 0 && (FULL || c * 16 < d);
          cp_async16(to + k_at<DK>(r, c), kp + (FULL || on ? r * d + c * 16 : 0), on);
        }
#pragma unroll
        for (int x = 0; x < VC / 4; ++x) {
          const int q = lane + 32 * x, r = q / (VC / 2), c = q - r * (VC / 2);
          const bool on = at >= 0 && (FULL || c * 16 < dv);
          cp_async16(to + 16 * Cfg::KP + v_at<VC>(r, c), vp + (FULL || on ? r * dv + c * 16 : 0), on);
        }
      }
      if ((i & 15) == 0) {
        ask_scale();
        if (NT > 3 || i > 0) store_scale(2 * i);         // (32 rows leave no registers for it to wait in)
      }
    }
    cp_async_commit();
  };

  ask_page(0);

  float f[NT][2], m[NT][2], l[NT][2], o[NT][MT][4];      // of the lane's columns 2t, 2t + 1

  // The sums of the warps joined (common maximum, scaled sums in warp order) and written: the item's result, or this CTA's
  // part of it.  `free`: the stage of the segment's last block, where every warp puts its O.
  auto join = [&](const KvSegment& s, int free) {
    float* s_o = reinterpret_cast<float*>(smem + (size_t)free * Cfg::STAGE);          // of warp 0
    constexpr int WARP_O = STAGES * Cfg::STAGE / 4;                                    // floats from one warp's to the next
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], x);
        if (g == 0) {
          s_m[warp * ROWS + nt * 8 + 2 * t + j] = m[nt][j];
          s_l[warp * ROWS + nt * 8 + 2 * t + j] = l[nt][j];
        }
      }
    __syncthreads();
    if (tid < ROWS) {
      // a row's maximum and sum over the warps, and every warp's weight in place of its maximum
      float mk[KV_WARPS], lk[KV_WARPS], top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int k = 0; k < KV_WARPS; ++k) { mk[k] = s_m[k * ROWS + tid]; lk[k] = s_l[k * ROWS + tid]; top = fmaxf(top, mk[k]); }
#pragma unroll
      for (int k = 0; k < KV_WARPS; ++k) {
        const float w = mk[k] == -INFINITY ? (lk[k] == 0.f ? 0.f : 1.f) : fast_exp2(mk[k] - top);    // (l NaN without a maximum: kept)
        s_m[k * ROWS + tid] = w;
        sum += lk[k] * w;
      }
      s_tot[tid] = make_float2(top, sum);
    }
    __syncthreads();
    const bool whole = s.u0 == 0 && s.u1 == s.units;
    const int slot = 2 * blockIdx.x + (s.u0 > 0 ? 0 : 1);
#pragma unroll
    for (int pass = 0; pass < NT / JOIN; ++pass) {
      if (pass) __syncthreads();                           // O of the pass before has been read
#pragma unroll
      for (int n = 0; n < JOIN; ++n) {
        const int nt = pass * JOIN + n;
        const float2 w = *reinterpret_cast<const float2*>(s_m + warp * ROWS + nt * 8 + 2 * t);
#pragma unroll
        for (int jj = 0; jj < MT; ++jj)
#pragma unroll
          for (int c = 0; c < 4; ++c) s_o[warp * WARP_O + ((n * MT + jj) * 4 + c) * 32 + lane] = o[nt][jj][c] * (c & 1 ? w.y : w.x);
      }
      __syncthreads();
      // thread = 4 neighbouring dims of a row
#pragma unroll 1
      for (int x = tid; x < JOIN * 8 * DV / 4; x += KV_WARPS * 32) {
        constexpr int CH = VC < 16 ? VC : 16;              // bytes of one chunk
        const int c8 = x / (DV / 4), dim = (x - c8 * (DV / 4)) * 4, chunk = dim / (8 * CH), in = dim - chunk * 8 * CH;
        const int gg = in / CH, byte = in - gg * CH + chunk * CH, col = pass * JOIN * 8 + c8, row = s.row0 + col, i = row / p.G;
        if (i >= p.S) break;                               // (rows go up with x)
        const float* src = s_o + ((c8 >> 3) * MT * 4 + (byte >> 1) * 4 + (c8 & 1)) * 32 + gg * 4 + ((c8 & 7) >> 1);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KV_WARPS; ++k)
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] += src[k * WARP_O + (c >> 1) * 128 + (c & 1) * 64];
        float2 tot = s_tot[col];
        if (whole) {
          const int hq = s.h * p.G + row - i * p.G;
          if (p.sink) {
            const float sk = p.sink[hq] * kLog2e, up = fmaxf(tot.x, sk), z = tot.x == -INFINITY ? 1.f : fast_exp2(tot.x - up);
            tot.y = tot.y * z + (sk == -INFINITY ? 0.f : fast_exp2(sk - up));
            v[0] *= z; v[1] *= z; v[2] *= z; v[3] *= z;
            tot.x = up;
          }
          const float inv = tot.y == 0.f ? 0.f : 1.f / tot.y;
          if (dim == 0) p.lse[((int64_t)s.b * p.Hq + hq) * p.S + i] = tot.y == 0.f ? -INFINITY : (tot.x + log2f(tot.y)) * kLn2;
          if (FULL || dim < dv) {
            const uint2 z = p.bf16 ? make_uint2(pack2<true>(v[0] * inv, v[1] * inv), pack2<true>(v[2] * inv, v[3] * inv))
                                   : make_uint2(pack2<false>(v[0] * inv, v[1] * inv), pack2<false>(v[2] * inv, v[3] * inv));
            *reinterpret_cast<uint2*>(p.o + (((int64_t)s.b * p.S + i) * p.Hq + hq) * dv + dim) = z;
          }
        } else {
          *reinterpret_cast<float4*>(p.part_o + ((size_t)slot * ROWS + col) * DV + dim) = make_float4(v[0], v[1], v[2], v[3]);
          if (dim == 0) *reinterpret_cast<float2*>(p.part_ml + ((size_t)slot * ROWS + col) * 2) = tot;
        }
      }
    }
  };

  KvSegment seg;
  int seg_end = INT_MIN, lo_max = 0, hi_min = 0, stage = 0, free_stage = 0;
#pragma unroll 1
  for (int i = 1 - STAGES; i <= n_units; ++i) {
    if (i >= 0 && i < n_units) {
      cp_async_wait<STAGES - 2>();
      __syncwarp();                                    // block i is here, and every lane is done with block i - 1
    }
    // (the first item's turn comes ahead of its data)
    const bool turn = i == seg_end || i == 1 - STAGES;
    KvSegment last;
    uint4 x[DK][2];
    if (turn) {
      // the next item's queries (row g of tile `warp`) are on their way while the last one's sums are joined
      last = seg;
      const int at = max(i, 0);
      if ((at + STAGES - 2) >> 4 == at >> 4) seg = ahead.of_lane(2 * (at & 15));      // (looked up with the units of its round)
      else if (at < n_units) seg = segment(u_begin + at);
      const int row = seg.row0 + warp * 8 + g, qi = row / p.G;
      const bool on = warp < NT && i < n_units && qi < p.S;
      const uint16_t* src = p.q + seg.b * p.qs[0] + qi * p.qs[1] + ((int64_t)seg.h * p.G + row - qi * p.G) * p.qs[2];
#pragma unroll
      for (int c = 0; c < DK; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int at = (t + 4 * c) * 16 + j * 8;
          x[c][j] = make_uint4(0, 0, 0, 0);
          if (on && (FULL || at < d)) x[c][j] = __ldg(reinterpret_cast<const uint4*>(src + at));
        }
      if (i > 0) join(last, free_stage);
      if (i == n_units) break;
      if (i > 0) __syncthreads();                          // the join's reads of O, m and l
    }
    fetch(i + STAGES - 1, free_stage);
    free_stage = free_stage + 1 == STAGES ? 0 : free_stage + 1;
    if (turn) {
      seg_end = max(i, 0) + seg.u1 - seg.u0;
      if (tid < ROWS) {
        const int row = (seg.row0 + tid) / p.G;
        int lo, hi;
        row_range(p, seg.r, row, lo, hi);
        if (row >= p.S) { lo = 0; hi = INT_MAX; }          // (a column of zeros that nobody reads)
        s_lim[tid] = make_int2(lo, hi);
      }
      if (warp < NT) {
        // bf16 -> fp16: the row's largest exponent goes into its scale, and fp16 holds q 2^-e to 2^-24 of the row's largest value
        float scale = 1.f;
        if (p.bf16) {
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
          const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
          scale = __uint_as_float((uint32_t)e << 23);
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
          uint2* to = s_q + ((warp * DK + c) * 4) * 32 + lane;
          to[0] = make_uint2(x[c][0].x, x[c][0].y); to[32] = make_uint2(x[c][0].z, x[c][0].w);
          to[64] = make_uint2(x[c][1].x, x[c][1].y); to[96] = make_uint2(x[c][1].z, x[c][1].w);
        }
        if (t == 0) s_f[warp * 8 + g] = scale * p.scale_log2;
      }
      if (NT <= 3 && i < 0) store_scale(0);
      __syncthreads();                                    // s_lim, s_q, s_f
      lo_max = 0; hi_min = INT_MAX;
      if (lane < ROWS) { lo_max = s_lim[lane].x; hi_min = s_lim[lane].y; }
      lo_max = __reduce_max_sync(0xffffffffu, lo_max);
      hi_min = __reduce_min_sync(0xffffffffu, hi_min);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < 2; ++j) { f[nt][j] = s_f[nt * 8 + 2 * t + j]; m[nt][j] = -INFINITY; l[nt][j] = 0.f; }
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][j][c] = 0.f;
      }
    }
    if (i < 0) continue;
    const unsigned char* from = smem + (warp * STAGES + stage) * Cfg::STAGE;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    const int k0 = seg.key0 + KV_BLOCK * warp + (i - seg_end + seg.u1 - seg.u0) * KV_UNIT;

    float s[NT][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[nt][hh][c] = 0.f;
#pragma unroll 1
    for (int c = 0; c < DK; ++c) {
      uint4 x[2][2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        x[hh][0] = *reinterpret_cast<const uint4*>(from + hh * Cfg::GROUP + k_at<DK>(g, t + 4 * c));
        x[hh][1] = *reinterpret_cast<const uint4*>(from + hh * Cfg::GROUP + k_at<DK>(g + 8, t + 4 * c));
      }
      const uint2* q = s_q + c * 128 + lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t fr[2][4];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const uint32_t a = j == 0 ? x[hh][0].x : (j == 1 ? x[hh][0].y : (j == 2 ? x[hh][0].z : x[hh][0].w));
          const uint32_t z = j == 0 ? x[hh][1].x : (j == 1 ? x[hh][1].y : (j == 2 ? x[hh][1].z : x[hh][1].w));
          from_payload4<INT8>(a, fr[hh][0], fr[hh][2]);
          from_payload4<INT8>(z, fr[hh][1], fr[hh][3]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint2 y = q[nt * DK * 128 + j * 32];
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) mma(s[nt][hh], fr[hh], y.x, y.y);
        }
      }
    }
    const float4 i0 = info[(2 * i) & (KV_INFO - 1)], i1 = info[(2 * i + 1) & (KV_INFO - 1)];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float a = f[nt][j] * i0.x, z = f[nt][j] * i1.x;
        s[nt][0][j] = s[nt][0][j] * a + i0.y; s[nt][0][2 + j] = s[nt][0][2 + j] * a + i0.y;
        s[nt][1][j] = s[nt][1][j] * z + i1.y; s[nt][1][2 + j] = s[nt][1][2 + j] * z + i1.y;
      }
    uint32_t hidden = 0;                                   // bit nt * 8 + hh * 4 + q of a score that its row does not see
    const bool cut = k0 < lo_max || k0 + KV_BLOCK > hi_min;
    if (cut) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int2 lim = s_lim[nt * 8 + 2 * t + j];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int key = k0 + g + 8 * q;
            if (key < lim.x || key >= lim.y) {
              s[nt][q >> 1][(q & 1) * 2 + j] = -INFINITY;
              hidden |= 1u << (nt * 8 + (q >> 1) * 4 + (q & 1) * 2 + j);
            }
          }
        }
    }
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        grow |= fmaxf(fmax3(s[nt][0][j], s[nt][0][2 + j], s[nt][1][j]), s[nt][1][2 + j]) > m[nt][j] + 15.f;
    // m is kept 7 below the running maximum and lags: it moves where a score is more than 15 above it.  p is at most 2^15, and
    // fp16 keeps its relative precision down to 2^-21 of the largest
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = fmaxf(fmax3(s[nt][0][j], s[nt][0][2 + j], s[nt][1][j]), s[nt][1][2 + j]);
#pragma unroll
          for (int y = 4; y < 32; y <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, y));
          x = fmaxf(x - 7.f, m[nt][j]);
          const float w = x == -INFINITY ? 1.f : fast_exp2(m[nt][j] - x);
          m[nt][j] = x;
          l[nt][j] *= w;
#pragma unroll
          for (int jj = 0; jj < MT; ++jj) { o[nt][jj][j] *= w; o[nt][jj][2 + j] *= w; }
        }
    }
    uint32_t pb[2][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float e[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) e[q] = fast_exp2(s[nt][hh][q] - (q & 1 ? m1 : m0));
        l[nt][0] += (e[0] + e[2]) * (hh ? i1.z : i0.z);
        l[nt][1] += (e[1] + e[3]) * (hh ? i1.z : i0.z);
        pb[hh][nt][0] = movmatrix_trans(pack2<false>(e[0], e[1]));
        pb[hh][nt][1] = movmatrix_trans(pack2<false>(e[2], e[3]));
      }
    }
#pragma unroll 1
    for (int hh = 0; hh < 2; ++hh) {
      uint32_t vc[4][VW];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = 2 * t + (x & 1) + (x >> 1) * 8;
        const unsigned char* at = from + hh * Cfg::GROUP + 16 * Cfg::KP;
        if constexpr (VC == 8) {
          const uint2 v = *reinterpret_cast<const uint2*>(at + v_at<VC>(r, g >> 1) + (g & 1) * 8);
          vc[x][0] = v.x; vc[x][1] = v.y;
        } else {
#pragma unroll
          for (int c = 0; c < VC / 16; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(at + v_at<VC>(r, g + 8 * c));
            vc[x][4 * c] = v.x; vc[x][4 * c + 1] = v.y; vc[x][4 * c + 2] = v.z; vc[x][4 * c + 3] = v.w;
          }
        }
      }
      if (!INT8 && cut) {
        // A NaN among values that a row does not see (slots behind the sequence hold whatever was there) must stay out of
        // that row, and 0 * NaN would not: where a block that some row sees in part holds one, the NaNs are multiplied
        // apart, as ones, with what every row sees.
        uint32_t found = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int c = 0; c < VW; ++c) found |= nan_bytes(vc[x][c]);
        if (__any_sync(0xffffffffu, found != 0)) {
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
                float w[4], seen[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < 4; ++q) w[q] = hidden >> (nt * 8 + hh * 4 + q) & 1u ? 0.f : 1.f;
                mma(seen, fr, movmatrix_trans(pack2<false>(w[0], w[1])), movmatrix_trans(pack2<false>(w[2], w[3])));
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
          for (int nt = 0; nt < NT; ++nt) mma(o[nt][2 * c + half], fr, pb[0][nt][0], pb[0][nt][1]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) { pb[0][nt][0] = pb[1][nt][0]; pb[0][nt][1] = pb[1][nt][1]; }
    }
  }
}

// One CTA = one query row (of a kv head's rows) of one item; it joins the parts when the item was cut, which lie in
// consecutive CTAs' slots.  Where the item was cut follows from the lengths, which are there before the parts are.  Every
// warp computes all parts' weights, a lane each.  ONE: a row is a warp's (many rows of few parts), else a CTA's, whose
// warps take the parts in turn and are joined in order.
template <int DV, int ROWS, bool ONE>
__global__ void __launch_bounds__(128) kv_attn_merge_kernel(const __grid_constant__ KvAttnParams p) {
  constexpr int PER = DV / 32, AHEAD = 4, STEP = ONE ? 1 : 4;
  __shared__ float s_v[4][DV];
  __shared__ int s_sum[2][4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.z, h = blockIdx.y, row = ONE ? blockIdx.x * 4 + warp : blockIdx.x;
  const int first = ONE ? 0 : warp;                       // of the parts of this warp
  const int items = p.g.Hkv * p.row_tiles, mine = kv_units(kv_range(p, b));
  int before = 0, all = 0;
  for (int x = threadIdx.x; x < p.B; x += 128) {
    const int n = kv_units(kv_range(p, x)) * items;
    all += n;
    before += x < b ? n : 0;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) { all += __shfl_xor_sync(0xffffffffu, all, o); before += __shfl_xor_sync(0xffffffffu, before, o); }
  if (lane == 0) { s_sum[0][warp] = all; s_sum[1][warp] = before; }
  __syncthreads();
  const KvDeal deal(p.n_cta, s_sum[0][0] + s_sum[0][1] + s_sum[0][2] + s_sum[0][3], p.B * items);
  before = s_sum[1][0] + s_sum[1][1] + s_sum[1][2] + s_sum[1][3];
  const int tile = row / ROWS, in_tile = row - tile * ROWS;
  const int s0 = before + b * items * deal.extra + (h * p.row_tiles + min(tile, p.row_tiles - 1)) * (mine + deal.extra);
  const int c0 = deal.cta_of(s0), c1 = deal.cta_of(s0 + mine - 1);
  grid_dep_wait();
  if (c0 == c1 || row >= p.S * p.G) return;               // done by one CTA; no row
  auto slot = [&](int c) { return (size_t)(2 * c + (c == c0 ? 1 : 0)) * ROWS + in_tile; };
  auto get_ml = [&](int c) {
    return c <= c1 ? __ldcg(reinterpret_cast<const float2*>(p.part_ml) + slot(c)) : make_float2(-INFINITY, 0.f);
  };
  float y[AHEAD][PER];
  auto get_o = [&](int c) {                              // AHEAD parts of this warp, from c on
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const float* src = p.part_o + slot(c + STEP * a) * DV + lane * PER;
#pragma unroll
      for (int e = 0; e < PER; ++e) y[a][e] = 0.f;
      if (c + STEP * a > c1) continue;
      if constexpr (PER == 2) { const float2 q = __ldcg(reinterpret_cast<const float2*>(src)); y[a][0] = q.x; y[a][1] = q.y; }
      else {
#pragma unroll
        for (int e = 0; e < PER; e += 4) {
          const float4 q = __ldcg(reinterpret_cast<const float4*>(src + e));
          y[a][e] = q.x; y[a][e + 1] = q.y; y[a][e + 2] = q.z; y[a][e + 3] = q.w;
        }
      }
    }
  };
  float2 ml = get_ml(c0 + lane);
  get_o(c0 + first);
  const int i = row / p.G, hq = h * p.G + row - i * p.G;
  const float sk = p.sink ? p.sink[hq] * kLog2e : -INFINITY;
  float top = fmaxf(sk, ml.x);
  for (int c = c0 + 32 + lane; c <= c1; c += 32) top = fmaxf(top, get_ml(c).x);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = 0.f, v[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) v[x] = 0.f;
  for (int base = c0; base <= c1; base += 32) {
    if (base > c0) ml = get_ml(base + lane);
    const float w_mine = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - top);    // (l NaN without a maximum: kept)
    sum += ml.y * w_mine;
    for (int x0 = first; x0 < 32 && base + x0 <= c1; x0 += STEP * AHEAD) {
      if (base + x0 > c0 + first) get_o(base + x0);
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const float w = __shfl_sync(0xffffffffu, w_mine, x0 + STEP * a);
#pragma unroll
        for (int e = 0; e < PER; ++e) v[e] += base + x0 + STEP * a <= c1 ? w * y[a][e] : 0.f;
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (sk != -INFINITY) sum += fast_exp2(sk - top);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (lane == 0 && (ONE || warp == 0)) p.lse[((int64_t)b * p.Hq + hq) * p.S + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  uint16_t* out = p.o + (((int64_t)b * p.S + i) * p.Hq + hq) * p.dv;
  if constexpr (ONE) {
    if (lane * PER < p.dv)
#pragma unroll
      for (int x = 0; x < PER; x += 2)
        *reinterpret_cast<uint32_t*>(out + lane * PER + x) = p.bf16 ? pack2<true>(v[x] * inv, v[x + 1] * inv) : pack2<false>(v[x] * inv, v[x + 1] * inv);
  } else {
#pragma unroll
    for (int x = 0; x < PER; ++x) s_v[warp][lane * PER + x] = v[x];
    __syncthreads();
    for (int dim = threadIdx.x * 2; dim < p.dv; dim += 256) {
      const float x = (s_v[0][dim] + s_v[1][dim] + s_v[2][dim] + s_v[3][dim]) * inv;
      const float y2 = (s_v[0][dim + 1] + s_v[1][dim + 1] + s_v[2][dim + 1] + s_v[3][dim + 1]) * inv;
      *reinterpret_cast<uint32_t*>(out + dim) = p.bf16 ? pack2<true>(x, y2) : pack2<false>(x, y2);
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int sm_count();
int kv_geometry(const fm_kv_cache* c, const fm_kv_args* a, KvGeom* g);

constexpr int KV_MAX_B = 1024;                      // first units of the sequences are kept in shared memory

template <class Cfg>
static size_t kv_smem(int B) { return Cfg::FIXED + (size_t)std::max(B + 1, KV_WARPS * 33) * 4; }        // with the first units of the sequences
// CTAs that an SM holds (228 KB, 1 KB of each the system's).  More would run behind the others, with an equal share of the work: 1024
// sequences of 64 keys, d = 64, 92 us with a fourth CTA that does not fit, 72 us without.
template <class Cfg>
static int kv_ctas(int B) {
  static_assert(Cfg::CTAS > 1 || Cfg::FIXED + (KV_MAX_B + 1) * 4 <= 227 * 1024, "one CTA always fits");
  return (kv_smem<Cfg>(B) + 1024) * Cfg::CTAS <= 228 * 1024 ? Cfg::CTAS : Cfg::CTAS - 1;
}

struct KvAttnPlan { int vc, nt, n_cta; size_t bytes; };
static KvAttnPlan kv_attn_plan(const fm_kv_cache* c, const fm_kv_args* a) {
  KvAttnPlan pl;
  const int64_t rows = (int64_t)a->S * (a->Hq / c->Hkv);
  pl.vc = c->dv <= 64 && c->d <= 64 ? 8 : (c->dv <= 128 ? 16 : 32);
  pl.nt = rows <= 8 || pl.vc == 32 ? 1 : (rows <= 16 || c->d > 128 ? 2 : (rows <= 24 ? 3 : 4));
  pl.n_cta = sm_count() * (pl.vc > 16 ? kv_ctas<KvCfg<4, 32, 1>>(a->B) : c->d > 128 ? (pl.nt == 1 ? kv_ctas<KvCfg<3, 16, 1>>(a->B) : kv_ctas<KvCfg<3, 16, 2>>(a->B))
             : pl.vc == 16 ? (pl.nt == 1 ? kv_ctas<KvCfg<2, 16, 1>>(a->B) : pl.nt == 2 ? kv_ctas<KvCfg<2, 16, 2>>(a->B) : pl.nt == 3 ? kv_ctas<KvCfg<2, 16, 3>>(a->B) : kv_ctas<KvCfg<2, 16, 4>>(a->B))
                           : (pl.nt == 1 ? kv_ctas<KvCfg<1, 8, 1>>(a->B) : pl.nt == 2 ? kv_ctas<KvCfg<1, 8, 2>>(a->B) : pl.nt == 3 ? kv_ctas<KvCfg<1, 8, 3>>(a->B) : kv_ctas<KvCfg<1, 8, 4>>(a->B)));
  pl.bytes = (size_t)2 * pl.n_cta * pl.nt * 8 * (8 * pl.vc + 2) * sizeof(float);
  return pl;
}

template <int DK, int VC, int NT, bool INT8, bool FULL>
static int launch_kv_attn(const KvAttnParams& p, cudaStream_t s) {
  using Cfg = KvCfg<DK, VC, NT>;
  auto kern = kv_attn_kernel<DK, VC, NT, INT8, FULL>;
  static std::atomic<uint64_t> done{0};
  FM_CUDA_TRY(allow_smem(kern, (int)kv_smem<Cfg>(KV_MAX_B), done));
  kern<<<p.n_cta, KV_WARPS * 32, kv_smem<Cfg>(p.B), s>>>(p);
  count_launches(1);
  FM_CUDA_TRY(cudaGetLastError());
  // (a row of up to 8 parts is one warp's)
  const int rows = p.S * p.G;
  if ((int64_t)p.B * p.g.Hkv * p.row_tiles * 8 >= p.n_cta)
    FM_CUDA_TRY(launch_dependent(kv_attn_merge_kernel<8 * VC, 8 * NT, true>, dim3((rows + 3) / 4, p.g.Hkv, p.B), dim3(128), 0, s, p));
  else
    FM_CUDA_TRY(launch_dependent(kv_attn_merge_kernel<8 * VC, 8 * NT, false>, dim3(rows, p.g.Hkv, p.B), dim3(128), 0, s, p));
  count_launches(1);
  return FM_OK;
}

template <int DK, int VC, bool INT8, bool FULL>
static int launch_kv_attn_rows(const KvAttnParams& p, int nt, cudaStream_t s) {
  if (nt == 1 || VC > 16) return launch_kv_attn<DK, VC, 1, INT8, FULL>(p, s);
  if constexpr (VC <= 16) {
    if (nt == 2 || DK > 2) return launch_kv_attn<DK, VC, 2, INT8, FULL>(p, s);
    if constexpr (DK <= 2) return nt == 3 ? launch_kv_attn<DK, VC, 3, INT8, FULL>(p, s) : launch_kv_attn<DK, VC, 4, INT8, FULL>(p, s);
  }
  return FM_ERR_UNSUPPORTED;
}

template <bool INT8>
static int dispatch_kv_attn(const KvAttnParams& p, const KvAttnPlan& pl, cudaStream_t s) {
  if (pl.vc == 32) return launch_kv_attn_rows<4, 32, INT8, true>(p, pl.nt, s);
  if (p.d == 192) return launch_kv_attn_rows<3, 16, INT8, true>(p, pl.nt, s);
  if (pl.vc == 16) return p.d == 128 && p.dv == 128 ? launch_kv_attn_rows<2, 16, INT8, true>(p, pl.nt, s) : launch_kv_attn_rows<2, 16, INT8, false>(p, pl.nt, s);
  return p.d == 64 && p.dv == 64 ? launch_kv_attn_rows<1, 8, INT8, true>(p, pl.nt, s) : launch_kv_attn_rows<1, 8, INT8, false>(p, pl.nt, s);
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
  FM_REQUIRE(rows < 1 << 30 && (units + 1) * tiles <= (INT_MAX - 1) / c->Hkv / a->B, FM_ERR_UNSUPPORTED, "fm_kv_attention: too many rows and keys for one call");
  FM_REQUIRE((int64_t)c->num_pages * c->Hkv * c->page_size / 16 < INT_MAX, FM_ERR_UNSUPPORTED, "fm_kv_attention: a cache of 2^31 groups of 16 tokens");
  FM_REQUIRE(a->workspace && a->workspace_bytes >= pl.bytes && ((uintptr_t)a->workspace & 15) == 0, FM_ERR_WORKSPACE,
             "fm_kv_attention: workspace of %zu bytes, %zu needed", a->workspace_bytes, pl.bytes);
  p.k = (const uint8_t*)c->k; p.v = (const uint8_t*)c->v; p.ks = c->k_scale; p.vs = c->v_scale;
  p.table = a->page_table; p.seqlens = a->seqlens; p.lengths = a->lengths;
  p.q = (const uint16_t*)a->q; p.o = (uint16_t*)a->o; p.lse = a->lse; p.sink = a->sink;
  p.B = a->B; p.S = a->S; p.Hq = a->Hq; p.G = (int)G; p.d = c->d; p.dv = c->dv;
  p.causal = a->causal; p.window = std::min(a->window, 1 << 30); p.bf16 = a->dtype == FM_DTYPE_BF16;
  p.row_tiles = (int)tiles;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.n_cta = pl.n_cta;
  p.part_o = (float*)a->workspace;
  p.part_ml = p.part_o + (size_t)2 * pl.n_cta * pl.nt * 8 * 8 * pl.vc;
  return c->dtype == FM_CACHE_INT8 ? dispatch_kv_attn<true>(p, pl, (cudaStream_t)stream) : dispatch_kv_attn<false>(p, pl, (cudaStream_t)stream);
}
