// Writing 16-bit keys and values into the 8-bit paged cache, and reading them back.
#include <algorithm>

#include "fm_kv_cache.cuh"

namespace fm {

struct KvWriteParams {
  KvGeom g;
  uint8_t* pay[2]; float* scale[2];
  const uint16_t* src[2];
  int64_t stride[2][3];
  int width[2];
  const int32_t* table; const int32_t* start; const int32_t* lengths;
  int B, S;
};

// How TEAM threads walk rows of `upr` units of 8 values: thread = unit `col` of rows row0, row0 + step, ..
struct RowWalk { int row0, step, col; };
template <int TEAM>
__device__ __forceinline__ RowWalk row_walk(int upr) {
  const unsigned tid = TEAM == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int step = TEAM / upr, row0 = tid / upr;
  return {row0 < step ? row0 : INT_MAX / 2, step, (int)tid - row0 * upr};
}

// One team (a CTA, or each of its warps) = one page of one kv head, K or V (2 * head + which), of the pages that the new tokens of
// sequence blockIdx.z reach.  It reads its tokens once, keeps them in registers while it finds the largest magnitude, and
// writes one byte for every two that it read.  Bound by HBM: 3 bytes a value.
// A page that held tokens before (the write starts inside it) keeps its scale or grows it; where it grows, the payload
// of the earlier tokens is rounded on the new grid.  Slots behind the last new token are left as they are.
// VEC = units of 8 values that a thread holds.
// Threads on an SM.  At these limits the CTAs' variants spill 60 to 196 bytes, and fewer threads with fewer spills take longer: pages of 64,
// us with these and with 1024 | 768 | 256 threads for 4 | 8 | 16 units: 4 x 8192 tokens, 8 heads, d = 64 (4 units) e4m3 20.8 / 26.1, int8 23.3 / 24.9; 2 x 8192,
// d = 128 (8 units) 19.2 / 19.7, 20.4 / 22.3; 4 heads, d = 256, pages of 128 (16 units) 25.8 / 32.5, 26.7 / 36.9.  64 registers for eight units spill less in
// int8 than in e4m3: with 1024 / 896 threads int8 20.9 / 22.0, e4m3 23.3 / 19.3.
constexpr int write_threads(bool int8, int vec) { return vec <= 4 ? 1280 : (vec > 8 ? 512 : (int8 ? 1024 : 896)); }
template <bool IS_BF16, bool INT8, int VEC, int THREADS, int TEAM>
__global__ void __launch_bounds__(THREADS, write_threads(INT8, VEC) / THREADS) kv_write_kernel(const __grid_constant__ KvWriteParams p) {
  constexpr int WARPS = TEAM / 32;
  __shared__ uint32_t s_max[WARPS];
  const int b = blockIdx.z, hw = TEAM == THREADS ? blockIdx.y : blockIdx.y * (THREADS / TEAM) + threadIdx.x / TEAM, which = hw & 1, h = hw >> 1, P = 1 << p.g.page_log2;
  if (THREADS > TEAM && h >= p.g.Hkv) return;
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
  const int start = p.start[b];
  // positions that are written: none before 0 or behind the page table (2^31 - 2^16 at most), however far the rows reach
  const int first = max(start, 0), last = (int)min((int64_t)start + n, (int64_t)p.g.cap) - 1;
  const int64_t base64 = (int64_t)((first >> p.g.page_log2) + blockIdx.x) << p.g.page_log2;
  if (last < first || base64 > last) return;
  const int base = (int)base64;
  const int page = kv_page(p.g, p.table + b * p.g.table_stride, base);
  if (page < 0) return;
  const int w = p.width[which];
  const RowWalk at = row_walk<TEAM>(w >> 3);
  const int lo = max(first - base, 0), hi = min(last - base + 1, P);       // slots [lo, hi) are new
  uint8_t* pay = p.pay[which] + ((size_t)page * p.g.Hkv + h) * P * w + at.col * 8;
  float* scale = p.scale[which] + (size_t)page * p.g.Hkv + h;
  const int64_t ss = p.stride[which][1];
  const uint16_t* src = p.src[which] + b * p.stride[which][0] + h * p.stride[which][2] + (base - start) * ss + at.col * 8;
  const float old = lo > 0 ? *scale : 0.f;
  uint4 x[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int row = lo + at.row0 + i * at.step;
    x[i] = row < hi ? __ldcs(reinterpret_cast<const uint4*>(src + row * ss)) : make_uint4(0, 0, 0, 0);
  }
  // the largest magnitude, as bits: of 16-bit floats these have the order of the values, infinities and NaN on top
  constexpr uint32_t INF = IS_BF16 ? 0x7f80u : 0x7c00u;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    top = __vmaxu2(top, __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu), __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu)));
  }
  top = max(top & 0xffffu, top >> 16);
  const int warp = threadIdx.x >> 5;
  auto largest = [&](uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (WARPS > 1) {
      if ((threadIdx.x & 31) == 0) s_max[warp] = v;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < WARPS; ++i) v = max(v, s_max[i]);
    }
    return v;
  };
  top = largest(top);
  const bool bad = top >= INF;
  if (bad) {
    // What is no number does not set the scale and has no payload: NaN in e4m3, 0 in int8, where the scale says it.
    top = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      uint32_t* v = reinterpret_cast<uint32_t*>(&x[i]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t l = v[c] & 0x7fffu, u = v[c] >> 16 & 0x7fffu;
        if (l < INF) top = max(top, l); else v[c] = (v[c] & 0xffff0000u) | (INT8 ? 0u : 0x7fffu);
        if (u < INF) top = max(top, u); else v[c] = (v[c] & 0xffffu) | (INT8 ? 0u : 0x7fff0000u);
      }
    }
    if constexpr (WARPS > 1) __syncthreads();
    top = largest(top);
  }
  int e = cache_exponent<INT8>(unpack2<IS_BF16>(top).x);
  const bool old_nan = INT8 && lo > 0 && !(old > 0.f);           // a NaN scale stays until the page is started again
  const int e_old = (int)(__float_as_uint(old) >> 23 & 0xff) - 127;
  if (lo > 0 && !old_nan) e = max(e, min(max(e_old, kCacheMinExp), kCacheMaxExp<INT8>));
  const float inv = exp2_int(-e);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int row = lo + at.row0 + i * at.step;
    if (row < hi) {
      const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint32_t r[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 f = unpack2<IS_BF16>(v[c]);
        r[c] = to_payload2<INT8>(f.x * inv, f.y * inv);
      }
      *reinterpret_cast<uint2*>(pay + row * w) = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
    }
  }
  if (lo > 0 && !old_nan && e > e_old) {
    const float f = exp2_int(max(e_old - e, -126));
    for (int row = at.row0; row < lo; row += at.step) {
      uint2* to = reinterpret_cast<uint2*>(pay + row * w);
      uint2 v = *to;
      float a[4];
      payload_f32<INT8>(v.x, a);
      v.x = to_payload2<INT8>(a[0] * f, a[1] * f) | to_payload2<INT8>(a[2] * f, a[3] * f) << 16;
      payload_f32<INT8>(v.y, a);
      v.y = to_payload2<INT8>(a[0] * f, a[1] * f) | to_payload2<INT8>(a[2] * f, a[3] * f) << 16;
      *to = v;
    }
  }
  // Every thread has read the old scale, so it can go: a CTA's barrier lies between, a warp's lanes have only exchanged their
  // magnitudes, which orders no memory.
  if constexpr (WARPS == 1) __syncwarp();
  if ((threadIdx.x & (TEAM - 1)) == 0) *scale = INT8 && (bad || old_nan) ? __uint_as_float(0x7fffffffu) : exp2_int(e);
}

struct KvReadParams {
  KvGeom g;
  const uint8_t* pay[2]; const float* scale[2];
  uint16_t* dst[2];
  int width[2];
  const int32_t* table; const int32_t* start; const int32_t* seqlens;
  int32_t* marks;                                                // [B, Hkv] (MARK)
  int B, S;
};

// dst[b, i, h, :] = the token at position start[b] + i, zeros where it has none.  One team (a CTA, or each of its warps) = the rows in one page of one kv
// head, K and V: the page and its scales are looked up once, and a thread has READ_ILP units of 8 bytes of each in flight.
// Bound by HBM: 3 bytes a value (2 x 8192 tokens of 8 heads, d = 128, 100 MB: e4m3 14.5 us, int8 16, 6.3 TB/s; CTAs of 256 threads 18.5 us).
// Eight CTAs to an SM at 64 registers and up to 20 bytes of spills; seven: e4m3 14.9, int8 15.6.
// MARK: for a dense forward, whose P V would take 0 * NaN into rows that do not see the token.  What is NaN comes as 0, and
// marks[b, h] says that there was some; kv_nan_kernel brings it to the rows that see it.
constexpr int READ_ILP = 4;
template <bool IS_BF16, bool INT8, int TEAM, bool MARK>
__global__ void __launch_bounds__(128, 8) kv_read_kernel(const __grid_constant__ KvReadParams p) {
  const int b = blockIdx.z, h = TEAM == 128 ? blockIdx.y : blockIdx.y * (128 / TEAM) + threadIdx.x / TEAM, P = 1 << p.g.page_log2;
  if (TEAM < 128 && h >= p.g.Hkv) return;
  const int64_t start = p.start[b], base = ((start >> p.g.page_log2) + blockIdx.x) << p.g.page_log2;      // (rounds down below 0 too)
  const int len = kv_len(p.g, p.seqlens[b]);
  if (base >= start + p.S) return;
  const int page = base >= 0 && base < len ? kv_page(p.g, p.table + b * p.g.table_stride, (int)base) : -1;
  const int lo = base < start ? (int)(start - base) : 0, hi = (int)min((int64_t)P, start + p.S - base);    // slots that are asked for
  const int valid = page >= 0 ? (int)min((int64_t)P, len - base) : 0;                                      // slots that hold tokens
  const size_t ph = (size_t)max(page, 0) * p.g.Hkv + h;
  const RowWalk at[2] = {row_walk<TEAM>(p.width[0] >> 3), row_walk<TEAM>(p.width[1] >> 3)};
  float scale[2];
  const uint8_t* pay[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    scale[x] = page >= 0 ? __ldg(p.scale[x] + ph) : 0.f;
    pay[x] = p.pay[x] + ph * P * p.width[x] + at[x].col * 8;
  }
  bool found = false;
  for (int row0 = lo; row0 < hi; row0 += READ_ILP * min(at[0].step, at[1].step)) {
    uint2 v[2][READ_ILP];
    const int upto = min(hi, row0 + READ_ILP * min(at[0].step, at[1].step));
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < READ_ILP; ++i) {
        const int row = row0 + at[x].row0 + i * at[x].step;
        v[x][i] = row < upto && row < valid ? __ldcs(reinterpret_cast<const uint2*>(pay[x] + row * p.width[x])) : make_uint2(0, 0);
      }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int64_t out_row = (int64_t)p.g.Hkv * p.width[x];
      uint16_t* dst = p.dst[x] + ((int64_t)b * p.S + (base - start)) * out_row + h * p.width[x] + at[x].col * 8;
#pragma unroll
      for (int i = 0; i < READ_ILP; ++i) {
        const int row = row0 + at[x].row0 + i * at[x].step;
        if (row >= upto) break;
        float a[4], c[4];
        if constexpr (MARK && !INT8) {
          const uint32_t n0 = nan_bytes(v[x][i].x), n1 = nan_bytes(v[x][i].y);
          if ((n0 | n1) != 0) {
            found = true;
            v[x][i].x &= ~((n0 >> 7) * 0xffu);
            v[x][i].y &= ~((n1 >> 7) * 0xffu);
          }
        }
        payload_f32<INT8>(v[x][i].x, a);
        payload_f32<INT8>(v[x][i].y, c);
        float sc = row < valid ? scale[x] : 0.f;                  // (a NaN scale is no token's)
        if constexpr (MARK) {
          if (sc != sc) { sc = 0.f; found = true; }               // (looked at here: the payload is asked for before the scale is there)
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[j] *= sc; c[j] *= sc;
          // the 8-bit grid reaches a little beyond fp16; NaN passes
          if (!IS_BF16) { if (fabsf(a[j]) > 65504.f) a[j] = copysignf(65504.f, a[j]); if (fabsf(c[j]) > 65504.f) c[j] = copysignf(65504.f, c[j]); }
        }
        *reinterpret_cast<uint4*>(dst + row * out_row) = make_uint4(pack2<IS_BF16>(a[0], a[1]), pack2<IS_BF16>(a[2], a[3]),
                                                                    pack2<IS_BF16>(c[0], c[1]), pack2<IS_BF16>(c[2], c[3]));
      }
    }
  }
  if (MARK && found) p.marks[(int64_t)b * p.g.Hkv + h] = 1;
}

// Column bounds that make a dense causal forward over the read-back tokens see what the cache's rows see.  Column c
// of sequence b holds position shift_b + c.  With `n` real query rows (of Sq) and rows counted from the first, position
// p is hidden from row i on: i >= n (no query), i >= p - p0 + window (out of the window), and everywhere when it is no
// token.  Causal: lower bound alone.
struct KvBoundsParams {
  KvGeom g;
  const int32_t* seqlens; const int32_t* lengths; const int32_t* table;
  int32_t* shift; int32_t* bounds; int32_t* marks;              // marks: zeroed, or NULL
  int B, Sq, cols, causal, window;
};
__global__ void __launch_bounds__(256) kv_bounds_kernel(const KvBoundsParams p) {
  const int b = blockIdx.y;
  const int c = blockIdx.x * 256 + threadIdx.x;
  const int len = kv_len(p.g, p.seqlens[b]);
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.Sq) : p.Sq;
  // the first row stands at len - n and, bottom-right aligned, sees the columns up to cols - Sq
  const int shift = len - n - (p.cols - p.Sq);
  if (c == 0) p.shift[b] = shift;
  if (p.marks && blockIdx.x == 0)
    for (int h = threadIdx.x; h < p.g.Hkv; h += 256) p.marks[(int64_t)b * p.g.Hkv + h] = 0;
  if (c >= p.cols) return;
  const int pos = shift + c;
  int end = 0;
  if (pos >= 0 && pos < len && kv_page(p.g, p.table + b * p.g.table_stride, pos) >= 0) {
    end = n;
    if (p.window > 0) end = (int)min((int64_t)end, (int64_t)pos - (len - n) + p.window);
  }
  end = max(end, 0);
  if (p.causal) p.bounds[(int64_t)b * p.cols + c] = end;
  else reinterpret_cast<int2*>(p.bounds)[(int64_t)b * p.cols + c] = make_int2(end, 0);
}

// NaN for the rows of a dense forward that see a token whose key or value is none (it got 0 in its place): the whole row and its
// lse where a key or a page's scale is NaN, the value's column where a value in e4m3 is.  And an lse of NaN for the other rows
// of NaN, those of a NaN query, which the dense forward leaves with -inf.
// One CTA = up to NAN_ROWS query rows of a sequence and kv head.  Nearly always there is no mark, and a CTA reads its rows' lse and leaves:
// the launch and one round trip to memory (512 rows of 16384 tokens, 32 / 8 heads: 160 -> 164 us; 40 of 300: 17.6 -> 19.5; 64 sequences, 25 of 512: 96 -> 102).  With a mark its warps walk the groups of 16 tokens that one of the rows sees, lanes
// side by side along the payload; tokens that all rows see, nearly all, cost no work per row.
struct KvNanParams {
  KvGeom g;
  const uint8_t* pay[2]; const float* scale[2];
  int width[2];
  const int32_t* table; const int32_t* seqlens; const int32_t* lengths; const int32_t* marks;
  uint16_t* o; float* lse;
  int B, S, Hq, G, causal, window;
};
constexpr int NAN_ROWS = 32, NAN_WORDS = 64;                     // (64 words of 4 values: 256 is the widest head)
template <bool IS_BF16, bool INT8>
__global__ void __launch_bounds__(256) kv_nan_kernel(const __grid_constant__ KvNanParams p) {
  __shared__ uint32_t s_cols[NAN_ROWS + 1][NAN_WORDS];           // 0x80 in the bytes of columns that are NaN; the last row: for every row
  __shared__ int s_row[NAN_ROWS + 1];                            // the whole row is
  constexpr uint32_t INF = IS_BF16 ? 0x7f80u : 0x7c00u;
  const int b = blockIdx.z, h = blockIdx.y, i0 = blockIdx.x * NAN_ROWS, rows = min(NAN_ROWS, p.S - i0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dv = p.width[1], words = dv / 4;
  const float nan = __uint_as_float(0x7fffffffu);
  grid_dep_wait();
  const int mark = __ldcg(p.marks + (int64_t)b * p.g.Hkv + h);
  if (lane < rows)
    for (int hq = h * p.G + warp; hq < (h + 1) * p.G; hq += 8) {
      float* lse = p.lse + ((int64_t)b * p.Hq + hq) * p.S + i0 + lane;
      if (__ldcg(lse) == -INFINITY && (__ldcg(p.o + (((int64_t)b * p.S + i0 + lane) * p.Hq + hq) * dv) & 0x7fffu) > INF) *lse = nan;
    }
  if (mark == 0) return;
  const int len = kv_len(p.g, p.seqlens[b]), n = p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
  const int live = min(rows, n - i0);                            // rows that are queries
  if (live <= 0) return;
  // keys [row_lo(r), row_hi(r)) of row r
  const int p0 = len - n + i0;
  auto row_lo = [&](int r) { return p.window > 0 ? max(p0 + r + 1 - p.window, 0) : 0; };
  auto row_hi = [&](int r) { return p.causal ? max(p0 + r + 1, 0) : len; };
  for (int x = tid; x < (NAN_ROWS + 1) * NAN_WORDS; x += 256) s_cols[x / NAN_WORDS][x % NAN_WORDS] = 0;
  if (tid <= NAN_ROWS) s_row[tid] = 0;
  __syncthreads();
  const int lo = row_lo(0), hi = row_hi(live - 1), all_lo = row_lo(live - 1), all_hi = row_hi(0);      // one row sees [lo, hi), all see [all_lo, all_hi)
  for (int g0 = (lo >> 4) + warp; g0 < (hi + 15) >> 4; g0 += 8) {
    const int page = kv_page(p.g, p.table + b * p.g.table_stride, g0 << 4);
    if (page < 0) continue;
    const size_t ph = (size_t)page * p.g.Hkv + h;
    const float ks = p.scale[0][ph], vs = p.scale[1][ph];
    const bool dead = ks != ks || vs != vs;
    if (INT8 && !dead) continue;
    const int slot = (g0 << 4) & ((1 << p.g.page_log2) - 1);
#pragma unroll 4
    for (int j = 0; j < 16; ++j) {
      const int pos = (g0 << 4) + j;
      const bool seen = pos >= lo && pos < hi;
      const uint8_t *k = p.pay[0] + ((ph << p.g.page_log2) + slot + j) * p.width[0], *v = p.pay[1] + ((ph << p.g.page_log2) + slot + j) * dv;
      uint32_t in_k = 0, in_v[NAN_WORDS / 32] = {};
      if (!INT8 && seen) {
#pragma unroll
        for (int c = 0; c < NAN_WORDS / 32; ++c) {
          const int w = lane + 32 * c;
          if (4 * w < p.width[0]) in_k |= nan_bytes(*reinterpret_cast<const uint32_t*>(k + 4 * w));
          if (w < words) in_v[c] = nan_bytes(*reinterpret_cast<const uint32_t*>(v + 4 * w));
        }
      }
      const bool whole = seen && (dead || __any_sync(0xffffffffu, in_k != 0));
      uint32_t any_v = 0;
#pragma unroll
      for (int c = 0; c < NAN_WORDS / 32; ++c) any_v |= in_v[c];
      if (!whole && !__any_sync(0xffffffffu, any_v != 0)) continue;
      const bool all = pos >= all_lo && pos < all_hi;
      for (int r = all ? NAN_ROWS : 0; r < (all ? NAN_ROWS + 1 : live); ++r) {
        if (!all && (pos < row_lo(r) || pos >= row_hi(r))) continue;
        if (whole && lane == 0) s_row[r] = 1;
#pragma unroll
        for (int c = 0; c < NAN_WORDS / 32; ++c)
          if (in_v[c]) atomicOr(&s_cols[r][lane + 32 * c], in_v[c]);
      }
    }
  }
  __syncthreads();
  for (int x = warp; x < live * p.G; x += 8) {
    const int r = x % live, i = i0 + r, hq = h * p.G + x / live;
    const bool whole = s_row[r] != 0 || s_row[NAN_ROWS] != 0;
    uint16_t* o = p.o + (((int64_t)b * p.S + i) * p.Hq + hq) * dv;
    for (int w = lane; w < words; w += 32) {
      const uint32_t cols = whole ? 0x80808080u : s_cols[r][w] | s_cols[NAN_ROWS][w];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (cols >> (8 * c + 7) & 1u) o[4 * w + c] = 0x7fffu;
    }
    if (whole && lane == 0) p.lse[((int64_t)b * p.Hq + hq) * p.S + i] = nan;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
static int page_log2_of(int page_size) {
  for (int l = 4; l <= 7; ++l)
    if (page_size == 1 << l) return l;
  return -1;
}

int kv_geometry(const fm_kv_cache* c, const fm_kv_args* a, KvGeom* g) {
  FM_REQUIRE(c && a, FM_ERR_INVALID_ARGUMENT, "kv cache: NULL argument");
  FM_REQUIRE(c->k && c->v && c->k_scale && c->v_scale, FM_ERR_INVALID_ARGUMENT, "kv cache: payload or scale is NULL");
  FM_REQUIRE(c->dtype == FM_CACHE_E4M3 || c->dtype == FM_CACHE_INT8, FM_ERR_INVALID_ARGUMENT, "kv cache: unknown payload type %d", c->dtype);
  FM_REQUIRE(a->dtype == FM_DTYPE_BF16 || a->dtype == FM_DTYPE_FP16, FM_ERR_INVALID_ARGUMENT, "kv cache: unknown dtype %d", a->dtype);
  FM_REQUIRE(c->num_pages > 0 && c->Hkv > 0, FM_ERR_INVALID_ARGUMENT, "kv cache: num_pages=%d, Hkv=%d", c->num_pages, c->Hkv);
  FM_REQUIRE(page_log2_of(c->page_size) > 0, FM_ERR_UNSUPPORTED, "kv cache: page_size %d is not 16, 32, 64 or 128", c->page_size);
  FM_REQUIRE(c->d > 0 && c->dv > 0 && c->d % 16 == 0 && c->dv % 16 == 0, FM_ERR_UNSUPPORTED,
             "kv cache: head dims %d / %d are not multiples of 16", c->d, c->dv);
  FM_REQUIRE((c->d <= 128 && c->dv <= 128) || (c->d == 192 && c->dv == 128) || (c->d == 256 && c->dv == 256), FM_ERR_UNSUPPORTED,
             "kv cache: head dims %d / %d are not served (<= 128, 192 / 128, 256 / 256)", c->d, c->dv);
  FM_REQUIRE(((uintptr_t)c->k & 15) == 0 && ((uintptr_t)c->v & 15) == 0, FM_ERR_INVALID_ARGUMENT, "kv cache: payload is not 16-byte aligned");
  FM_REQUIRE(a->B >= 0 && a->S >= 0 && a->max_pages >= 0, FM_ERR_INVALID_ARGUMENT, "kv cache: negative size");
  FM_REQUIRE(a->B <= 65535 && c->Hkv <= 32767, FM_ERR_UNSUPPORTED, "kv cache: more than 65535 sequences or 32767 heads");
  FM_REQUIRE((int64_t)a->max_pages * c->page_size < INT_MAX - 65536, FM_ERR_UNSUPPORTED, "kv cache: a page table of more than 2^31 positions");
  FM_REQUIRE(a->page_table || a->B == 0 || a->max_pages == 0, FM_ERR_INVALID_ARGUMENT, "kv cache: page_table is NULL");
  FM_REQUIRE(a->table_stride >= a->max_pages || a->B <= 1, FM_ERR_INVALID_ARGUMENT, "kv cache: table_stride below max_pages");
  g->num_pages = c->num_pages; g->page_log2 = page_log2_of(c->page_size); g->Hkv = c->Hkv;
  g->max_pages = a->max_pages; g->table_stride = a->table_stride;
  g->cap = a->max_pages * c->page_size;
  return FM_OK;
}

// Pages that S tokens reach wherever the first falls.
static unsigned pages_of(int S, int page_size) { return (unsigned)(((int64_t)S + page_size - 2) / page_size + 1); }

template <bool IS_BF16, bool INT8>
static int launch_write(const KvWriteParams& p, int page_size, int width_max, cudaStream_t s) {
  const unsigned pages = pages_of(p.S, page_size), heads = 2 * p.g.Hkv;
  const dim3 ctas(pages, heads, p.B), warps(pages, (heads + 3) / 4, p.B);
  const int upr = width_max / 8, rows = std::min(page_size, p.S);
  auto holds = [&](int threads, int vec) { return rows <= threads / upr * vec; };
  // A few tokens or small pages: a warp for each, so that nobody waits for a CTA's start and its barrier (4 x 8192 tokens of 64 values,
  // 8 heads, pages of 16: 20 us; a CTA of 256 threads each 74 us).  Else CTAs of 128 threads (64 tokens of 128 values, 2 x 8192 of them
  // with 8 heads: 19 us, 5.2 TB/s; 256 threads of four units 3 us more, 512 threads of two 10 us more), and of 256 where those do
  // not hold a page.
  if (holds(32, 1)) kv_write_kernel<IS_BF16, INT8, 1, 128, 32><<<warps, 128, 0, s>>>(p);
  else if (holds(32, 4)) kv_write_kernel<IS_BF16, INT8, 4, 128, 32><<<warps, 128, 0, s>>>(p);
  else if (holds(32, 8)) kv_write_kernel<IS_BF16, INT8, 8, 128, 32><<<warps, 128, 0, s>>>(p);
  else if (holds(128, 4)) kv_write_kernel<IS_BF16, INT8, 4, 128, 128><<<ctas, 128, 0, s>>>(p);
  else if (holds(128, 8)) kv_write_kernel<IS_BF16, INT8, 8, 128, 128><<<ctas, 128, 0, s>>>(p);
  else if (holds(256, 8)) kv_write_kernel<IS_BF16, INT8, 8, 256, 256><<<ctas, 256, 0, s>>>(p);
  else kv_write_kernel<IS_BF16, INT8, 16, 256, 256><<<ctas, 256, 0, s>>>(p);       // (128 tokens of 256 values: 4096 units; any width: 240 threads hold them)
  count_launches(1);
  FM_CUDA_TRY(cudaGetLastError());
  return FM_OK;
}

// A warp for a page's rows where two rounds of it are enough: 128 threads would not have READ_ILP units each (4 x 8192 tokens of 64
// values, pages of 16: 16 us; a CTA each 33 us).
template <bool IS_BF16, bool INT8, bool MARK>
static int launch_read(const KvReadParams& p, int page_size, cudaStream_t s) {
  const unsigned pages = pages_of(p.S, page_size);
  if (std::min(page_size, p.S) <= 32 / (std::max(p.width[0], p.width[1]) / 8) * 2 * READ_ILP)
    kv_read_kernel<IS_BF16, INT8, 32, MARK><<<dim3(pages, (p.g.Hkv + 3) / 4, p.B), 128, 0, s>>>(p);
  else
    kv_read_kernel<IS_BF16, INT8, 128, MARK><<<dim3(pages, p.g.Hkv, p.B), 128, 0, s>>>(p);
  count_launches(1);
  FM_CUDA_TRY(cudaGetLastError());
  return FM_OK;
}
template <bool MARK>
static int dispatch_read(const KvReadParams& p, bool bf, bool i8, int page_size, cudaStream_t s) {
  if (bf) return i8 ? launch_read<true, true, MARK>(p, page_size, s) : launch_read<true, false, MARK>(p, page_size, s);
  return i8 ? launch_read<false, true, MARK>(p, page_size, s) : launch_read<false, false, MARK>(p, page_size, s);
}

}  // namespace fm

using namespace fm;

extern "C" FM_API int64_t fm_kv_locate(const fm_kv_cache* c, const fm_kv_args* a, int b, int head, int64_t pos, int value) {
  KvGeom g;
  if (kv_geometry(c, a, &g) != FM_OK || b < 0 || b >= a->B || head < 0 || head >= c->Hkv || pos < INT_MIN || pos > INT_MAX) return -1;
  const int page = kv_page(g, a->page_table + (int64_t)b * g.table_stride, (int)pos);
  if (page < 0) return -1;
  return (((int64_t)page * c->Hkv + head) * c->page_size + (pos & (c->page_size - 1))) * (value ? c->dv : c->d);
}

extern "C" FM_API int fm_kv_write(const fm_kv_cache* c, const fm_kv_args* a, void* stream) {
  KvWriteParams p;
  const int rc = kv_geometry(c, a, &p.g);
  if (rc) return rc;
  if (a->B == 0 || a->S == 0 || a->max_pages == 0) return FM_OK;
  FM_REQUIRE(a->k && a->v && a->start, FM_ERR_INVALID_ARGUMENT, "fm_kv_write: key, value or start is NULL");
  FM_REQUIRE(((uintptr_t)a->k & 15) == 0 && ((uintptr_t)a->v & 15) == 0, FM_ERR_INVALID_ARGUMENT, "fm_kv_write: key or value is not 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    FM_REQUIRE(a->k_stride[i] % 8 == 0 && a->v_stride[i] % 8 == 0, FM_ERR_INVALID_ARGUMENT, "fm_kv_write: strides are not multiples of 8 elements");
  p.pay[0] = (uint8_t*)c->k; p.pay[1] = (uint8_t*)c->v; p.scale[0] = c->k_scale; p.scale[1] = c->v_scale;
  p.src[0] = (const uint16_t*)a->k; p.src[1] = (const uint16_t*)a->v;
  for (int i = 0; i < 3; ++i) { p.stride[0][i] = a->k_stride[i]; p.stride[1][i] = a->v_stride[i]; }
  p.width[0] = c->d; p.width[1] = c->dv;
  p.table = a->page_table; p.start = a->start; p.lengths = a->lengths;
  p.B = a->B; p.S = a->S;
  const bool bf = a->dtype == FM_DTYPE_BF16, i8 = c->dtype == FM_CACHE_INT8;
  const int wmax = c->d > c->dv ? c->d : c->dv;
  cudaStream_t s = (cudaStream_t)stream;
  if (bf) return i8 ? launch_write<true, true>(p, c->page_size, wmax, s) : launch_write<true, false>(p, c->page_size, wmax, s);
  return i8 ? launch_write<false, true>(p, c->page_size, wmax, s) : launch_write<false, false>(p, c->page_size, wmax, s);
}

extern "C" FM_API int fm_kv_read(const fm_kv_cache* c, const fm_kv_args* a, void* stream) {
  KvReadParams p;
  const int rc = kv_geometry(c, a, &p.g);
  if (rc) return rc;
  if (a->B == 0 || a->S == 0) return FM_OK;
  FM_REQUIRE(a->k_out && a->v_out && a->start && a->seqlens, FM_ERR_INVALID_ARGUMENT, "fm_kv_read: an output, start or seqlens is NULL");
  FM_REQUIRE(((uintptr_t)a->k_out & 15) == 0 && ((uintptr_t)a->v_out & 15) == 0, FM_ERR_INVALID_ARGUMENT, "fm_kv_read: an output is not 16-byte aligned");
  p.pay[0] = (const uint8_t*)c->k; p.pay[1] = (const uint8_t*)c->v; p.scale[0] = c->k_scale; p.scale[1] = c->v_scale;
  p.dst[0] = (uint16_t*)a->k_out; p.dst[1] = (uint16_t*)a->v_out;
  p.width[0] = c->d; p.width[1] = c->dv;
  p.table = a->page_table; p.start = a->start; p.seqlens = a->seqlens; p.marks = a->marks;
  p.B = a->B; p.S = a->S;
  const bool bf = a->dtype == FM_DTYPE_BF16, i8 = c->dtype == FM_CACHE_INT8;
  cudaStream_t s = (cudaStream_t)stream;
  return p.marks ? dispatch_read<true>(p, bf, i8, c->page_size, s) : dispatch_read<false>(p, bf, i8, c->page_size, s);
}

extern "C" FM_API int fm_kv_bounds(const fm_kv_cache* c, const fm_kv_args* a, int cols, int32_t* shift, int32_t* bounds, void* stream) {
  KvBoundsParams p;
  const int rc = kv_geometry(c, a, &p.g);
  if (rc) return rc;
  FM_REQUIRE(cols >= a->S && cols <= INT_MAX - 65536, FM_ERR_INVALID_ARGUMENT, "fm_kv_bounds: %d columns for %d query rows", cols, a->S);
  FM_REQUIRE(a->window >= 0 && (a->causal || a->window == 0), FM_ERR_INVALID_ARGUMENT, "fm_kv_bounds: window %d (causal %d)", a->window, a->causal);
  if (a->B == 0 || cols == 0) return FM_OK;
  FM_REQUIRE(a->seqlens && shift && bounds, FM_ERR_INVALID_ARGUMENT, "fm_kv_bounds: seqlens, shift or bounds is NULL");
  FM_REQUIRE(((uintptr_t)bounds & 7) == 0, FM_ERR_INVALID_ARGUMENT, "fm_kv_bounds: bounds is not 8-byte aligned");
  p.seqlens = a->seqlens; p.lengths = a->lengths; p.table = a->page_table;
  p.shift = shift; p.bounds = bounds; p.marks = a->marks;
  p.B = a->B; p.Sq = a->S; p.cols = cols; p.causal = a->causal; p.window = a->window;
  kv_bounds_kernel<<<dim3((unsigned)((cols + 255) / 256), a->B), 256, 0, (cudaStream_t)stream>>>(p);
  count_launches(1);
  FM_CUDA_TRY(cudaGetLastError());
  return FM_OK;
}

extern "C" FM_API int fm_kv_nan_rows(const fm_kv_cache* c, const fm_kv_args* a, void* stream) {
  KvNanParams p;
  const int rc = kv_geometry(c, a, &p.g);
  if (rc) return rc;
  FM_REQUIRE(a->Hq > 0 && a->Hq % c->Hkv == 0, FM_ERR_INVALID_ARGUMENT, "fm_kv_nan_rows: Hq=%d is no multiple of Hkv=%d", a->Hq, c->Hkv);
  FM_REQUIRE(a->window >= 0 && (a->causal || a->window == 0), FM_ERR_INVALID_ARGUMENT, "fm_kv_nan_rows: window %d (causal %d)", a->window, a->causal);
  if (a->B == 0 || a->S == 0) return FM_OK;
  FM_REQUIRE(a->o && a->lse && a->seqlens && a->marks, FM_ERR_INVALID_ARGUMENT, "fm_kv_nan_rows: o, lse, seqlens or marks is NULL");
  p.pay[0] = (const uint8_t*)c->k; p.pay[1] = (const uint8_t*)c->v; p.scale[0] = c->k_scale; p.scale[1] = c->v_scale;
  p.width[0] = c->d; p.width[1] = c->dv;
  p.table = a->page_table; p.seqlens = a->seqlens; p.lengths = a->lengths; p.marks = a->marks;
  p.o = (uint16_t*)a->o; p.lse = a->lse;
  p.B = a->B; p.S = a->S; p.Hq = a->Hq; p.G = a->Hq / c->Hkv;
  p.causal = a->causal; p.window = std::min(a->window, 1 << 30);
  const bool bf = a->dtype == FM_DTYPE_BF16, i8 = c->dtype == FM_CACHE_INT8;
  auto kern = bf ? (i8 ? kv_nan_kernel<true, true> : kv_nan_kernel<true, false>) : (i8 ? kv_nan_kernel<false, true> : kv_nan_kernel<false, false>);
  FM_CUDA_TRY(launch_dependent(kern, dim3((unsigned)((a->S + NAN_ROWS - 1) / NAN_ROWS), c->Hkv, a->B), dim3(256), 0, (cudaStream_t)stream, p));
  count_launches(1);
  return FM_OK;
}
