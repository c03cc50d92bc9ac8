// gb_chunk.cu -- attention of each sequence's new rows over a paged KV cache:
// row t of a sequence's n new rows (cpu.AttnDecode's arithmetic at one
// position each, backend/cpu/cpu.go:140-168) attends to positions
// [0, kv_len - n + t], through the page tables of gb_paged.cu.
//
//   o = sum_p softmax_p(scale q . k_p) v_p
//
// The G query heads of a KV head share its keys, so a unit of work packs them
// beside the tokens: packed row r = t * G + g of a sequence, a fixed number of
// packed rows and one KV head to a unit, its positions walked in tiles with a
// running maximum and sum (float32) for each row.
//
// Split of the work: the (unit, tile) pairs of all sequences form one line,
// cut into equal runs, one for each CTA of a grid that fills the GPU once. A
// unit cut by a run's end leaves its partial rows (maximum, sum, unnormalised
// output) in the workspace; the last CTA to arrive at that unit joins them in
// CTA order, so the result does not depend on which one that is. One rule
// serves one sequence decoding (a line of few units cut 148 ways), long
// prompts (whole units, cut only at the ends) and mixtures of both.
#include <math.h>

#include <algorithm>

#include <cuda_bf16.h>

#include "gb_device.cuh"
#include "gb_internal.h"

namespace {

struct ChunkArgs {
  gb_paged_chunk c;
  const void *q;
  void *out;
  long long ldq, ldo;
  int n_heads, G;
  float scale_log2;   // scale * log2(e): the softmax is taken in powers of two
  float *part;        // partial rows (part_slot)
  unsigned *counter;  // [CTAs], zero between launches
};

// ---- the line of work --------------------------------------------------------

// A sequence as the device data describe it, made safe: rows outside the
// call's, or a table shorter than kv_len, cannot lead outside the buffers.
struct Seq {
  int q0, n;      // first row, new rows
  int len0;       // positions before the new rows (may be negative: rows that see nothing)
  int cap;        // positions the sequence holds, at most what its table can name
};
GB_DEV Seq seq_of(const ChunkArgs &a, int b) {
  Seq s;
  const int lo = max(0, a.c.q_start[b]), hi = min(a.c.rows, a.c.q_start[b + 1]);
  const int len = a.c.kv_lens[b];
  s.q0 = lo;
  s.n = max(0, hi - lo);
  s.len0 = max(len, 0) - s.n;
  s.cap = min(max(len, 0), a.c.max_pages * a.c.page_size);
  return s;
}
// Positions that packed row r sees.
GB_DEV int visible(const Seq &s, int G, int r) { return max(0, min(s.cap, s.len0 + r / G + 1)); }

template <int RU, int KT>
struct Line {
  static GB_DEV int units(const Seq &s, int G) { return (int)(((long long)s.n * G + RU - 1) / RU); }
  // Tiles of unit u: up to the last position its last row sees; one where none is seen, so that the rows are written.
  static GB_DEV int tiles(const Seq &s, int G, int u) {
    const int last = (int)min((long long)s.n * G, (long long)(u + 1) * RU) - 1;
    return max(1, (visible(s, G, last) + KT - 1) / KT);
  }
  static GB_DEV long long seq_tiles(const ChunkArgs &a, int b) {
    const Seq s = seq_of(a, b);
    const int nu = units(s, a.G);
    long long t = 0;
    for (int u = 0; u < nu; u++) t += tiles(s, a.G, u);
    return t * a.c.n_kv;
  }
};

struct Plan {
  long long total, ctas;    // the line's length, and the CTAs it is cut for
  long long x0, x1;         // this CTA's run of it
  long long rem;            // x0's place within its sequence
  int b;
};

// Inclusive sum over the block's first NT threads (a multiple of 32, all of them calling).
template <int NT>
GB_DEV long long block_scan(long long v, long long *warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; w++) v += warp_sums[w];
  return v;
}

// Every CTA finds its run by itself: each thread counts the tiles of a
// sequence, and the sums of all of them are scanned. All NT threads call it.
template <int RU, int KT, int NT>
GB_DEV void make_plan(const ChunkArgs &a, Plan *plan, long long *warp_sums) {
  const int tid = threadIdx.x, batch = a.c.batch;
  long long total = 0, first = 0, scan = 0;
  for (int b0 = 0; b0 < batch; b0 += NT) {
    const long long v = b0 + tid < batch ? Line<RU, KT>::seq_tiles(a, b0 + tid) : 0;
    const long long s = block_scan<NT>(v, warp_sums);
    if (b0 == 0) first = v, scan = s;
    long long sum = 0;
    for (int w = 0; w < NT / 32; w++) sum += warp_sums[w];
    total += sum;
    __syncthreads();
  }
  // a line shorter than the grid goes to as many CTAs as it has tiles, so that no CTA amid a unit is without a piece
  const long long ctas = min((long long)gridDim.x, total), me = min((long long)blockIdx.x, ctas);
  const long long x0 = ctas ? total * me / ctas : 0, x1 = me < ctas ? total * (me + 1) / ctas : x0;
  long long base = 0;
  for (int b0 = 0; b0 < batch; b0 += NT) {
    long long v = first, s = scan;
    if (batch > NT) {
      v = b0 + tid < batch ? Line<RU, KT>::seq_tiles(a, b0 + tid) : 0;
      s = block_scan<NT>(v, warp_sums);
    }
    if (v && base + s - v <= x0 && x0 < base + s) {
      plan->b = b0 + tid;
      plan->rem = x0 - (base + s - v);
    }
    if (batch > NT) {
      for (int w = 0; w < NT / 32; w++) base += warp_sums[w];
      __syncthreads();
    }
  }
  if (tid == 0) plan->total = total, plan->ctas = ctas, plan->x0 = x0, plan->x1 = x1;
  __syncthreads();
}

// A walk over the pieces of this CTA's run: a piece is a unit's tiles [t0, t1).
template <int RU, int KT>
struct Walk {
  long long x, x1, total, ctas;
  int b, u, h, i;
  // the piece
  Seq s;
  int r0, nr;           // the unit's packed rows [r0, r0 + nr) of the sequence
  int head;             // its KV head
  int t0, t1, nt;       // tiles of the piece, and of the unit
  int c_first, c_last;  // CTAs that hold pieces of the unit

  GB_DEV void start(const ChunkArgs &a, const Plan &p) {
    x = p.x0, x1 = p.x1, total = p.total, ctas = p.ctas;
    if (x >= x1) return;
    b = p.b;
    s = seq_of(a, b);
    long long rem = p.rem;
    for (u = 0;; u++) {
      nt = Line<RU, KT>::tiles(s, a.G, u);
      const long long n = (long long)nt * a.c.n_kv;
      if (rem < n) break;
      rem -= n;
    }
    h = (int)(rem / nt);
    i = (int)(rem % nt);
  }
  GB_DEV bool next(const ChunkArgs &a) {
    if (x >= x1) return false;
    if (h == a.c.n_kv) {
      h = 0;
      if (++u == Line<RU, KT>::units(s, a.G)) {
        u = 0;
        do s = seq_of(a, ++b);
        while (s.n == 0);  // x < x1 <= total: a sequence with rows follows
      }
      nt = Line<RU, KT>::tiles(s, a.G, u);
    }
    r0 = u * RU;
    nr = (int)min((long long)RU, (long long)s.n * a.G - r0);
    head = h;
    t0 = i;
    t1 = (int)min((long long)nt, i + (x1 - x));
    const long long y0 = x - i, y1 = y0 + nt;  // the unit's place in the line
    c_first = (int)(((y0 + 1) * ctas - 1) / total);
    c_last = (int)((y1 * ctas - 1) / total);
    x += t1 - t0;
    i = 0;
    h++;
    return true;
  }
};

// The pool row of position p (in elements, for KV head h), -1 past the
// sequence's positions; a table entry outside the pool reads page 0, as the
// decode attention does.
GB_DEV long long pool_row(const ChunkArgs &a, const Seq &s, int b, int h, int p) {
  if (p >= s.cap) return -1;
  int phys = a.c.block_table[(long long)b * a.c.max_pages + p / a.c.page_size];
  if (phys < 0 || phys >= a.c.n_pages) phys = 0;
  return (((long long)phys * a.c.n_kv + h) * a.c.page_size + p % a.c.page_size) * a.c.head_dim;
}

// ---- partial rows ------------------------------------------------------------
// A CTA leaves at most two pieces for others to join: the one its run begins
// within (which = 0) and the one it begins and does not end (which = 1). Each
// has RU rows of kMaxHD floats, then their maxima, then their sums.
constexpr int kMaxHD = 128;
template <int RU>
GB_DEV float *part_slot(const ChunkArgs &a, int cta, int which) {
  return a.part + (size_t)(cta * 2 + which) * RU * (kMaxHD + 2);
}

GB_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int T>
GB_DEV void put4(void *out, long long i, float x, float y, float z, float w) {
  if constexpr (T == GB_F32) {
    *(float4 *)((float *)out + i) = make_float4(x, y, z, w);
  } else if constexpr (T == GB_F16) {
    const __half2 p = __floats2half2_rn(x, y), r = __floats2half2_rn(z, w);
    *(uint2 *)((uint16_t *)out + i) = make_uint2(*(const uint32_t *)&p, *(const uint32_t *)&r);
  } else {
    const __nv_bfloat162 p = __floats2bfloat162_rn(x, y), r = __floats2bfloat162_rn(z, w);
    *(uint2 *)((uint16_t *)out + i) = make_uint2(*(const uint32_t *)&p, *(const uint32_t *)&r);
  }
}

template <int T>
GB_DEV void ld4(const void *base, long long i, float *o) {
  if constexpr (T == GB_F32) {
    const float4 x = __ldg((const float4 *)((const float *)base + i));
    o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w;
  } else {
    const uint2 u = __ldg((const uint2 *)((const uint16_t *)base + i));
    const uint32_t w[2] = {u.x, u.y};
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if constexpr (T == GB_F16) {
        o[2 * e] = gb_half_to_float((uint16_t)w[e]);
        o[2 * e + 1] = gb_half_to_float((uint16_t)(w[e] >> 16));
      } else {
        o[2 * e] = __uint_as_float(w[e] << 16);
        o[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
      }
    }
  }
}

// One row by itself, by one warp: lane = position for the scores, lane = four
// dimensions for the sum over V. Taken for rows that came out with an infinity
// or NaN: a tile holds positions that some of its rows do not see, and their
// weight of zero does not stop a NaN or an infinity in V. Here the row meets
// nothing but its own positions, so what it shows is its own.
template <int T>
__device__ __noinline__ void redo_row(const ChunkArgs &a, const Seq s, int b, int head, int pr) {
  const int lane = threadIdx.x & 31, hd = a.c.head_dim, lim = visible(s, a.G, pr);
  const long long row = s.q0 + pr / a.G, hq = (long long)(head * a.G + pr % a.G) * hd;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < lim; p0 += 32) {
    const int p = p0 + lane;
    const long long at = p < lim ? pool_row(a, s, b, head, p) : -1;
    float sc = 0.f;
    if (at >= 0)
      for (int d = 0; d < hd; d += 4) {
        float x[4], y[4];
        ld4<T>(a.q, row * a.ldq + hq + d, x);
        ld4<T>(a.c.k_pool, at + d, y);
        sc = fmaf(x[0], y[0], fmaf(x[1], y[1], fmaf(x[2], y[2], fmaf(x[3], y[3], sc))));
      }
    sc = at >= 0 ? sc * a.scale_log2 : -INFINITY;
    const float mn = fmaxf(m, gb_warp_max(sc)), ms = mn == -INFINITY ? 0.f : mn, f = ex2(m - ms), e = ex2(sc - ms);
    l = fmaf(l, f, gb_warp_sum(e));
    m = mn;
    for (int k = 0; k < 4; k++) o[k] *= f;
    const int n = min(32, lim - p0);
    for (int j = 0; j < n; j++) {
      const float pj = __shfl_sync(0xffffffffu, e, j);
      const long long vj = __shfl_sync(0xffffffffu, at, j);
      if (4 * lane < hd && vj >= 0) {
        float v[4];
        ld4<T>(a.c.v_pool, vj + 4 * lane, v);
        for (int k = 0; k < 4; k++) o[k] = fmaf(pj, v[k], o[k]);
      }
    }
  }
  const float inv = lim > 0 ? 1.f / l : 0.f;
  if (4 * lane < hd) put4<T>(a.out, row * a.ldo + hq + 4 * lane, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}

// Joins the pieces of a unit, CTA by CTA: one warp to a row, four dimensions to a lane.
template <int T, int RU, typename W>
GB_DEV void join_pieces(const ChunkArgs &a, const W &w, int warp, int warps) {
  const int lane = threadIdx.x & 31, hd = a.c.head_dim;
  for (int r = warp; r < w.nr; r += warps) {
    float m = -INFINITY;
    for (int c = w.c_first + lane; c <= w.c_last; c += 32)
      m = fmaxf(m, __ldcg(part_slot<RU>(a, c, c == w.c_first) + RU * kMaxHD + r));
    m = gb_warp_max(m);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (m > -INFINITY)
      for (int c = w.c_first; c <= w.c_last; c++) {
        const float *p = part_slot<RU>(a, c, c == w.c_first);
        const float f = ex2(__ldcg(p + RU * kMaxHD + r) - m);
        l = fmaf(f, __ldcg(p + RU * (kMaxHD + 1) + r), l);
        const float4 v = __ldcg((const float4 *)(p + (size_t)r * kMaxHD) + lane);
        o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
      }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    if (4 * lane < hd) {
      const int pr = w.r0 + r;
      const long long at = (long long)(w.s.q0 + pr / a.G) * a.ldo + (long long)(w.head * a.G + pr % a.G) * hd + 4 * lane;
      put4<T>(a.out, at, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
    const bool odd = !isfinite(o.x * inv) || !isfinite(o.y * inv) || !isfinite(o.z * inv) || !isfinite(o.w * inv);
    if (__any_sync(0xffffffffu, 4 * lane < hd && odd)) redo_row<T>(a, w.s, w.b, w.head, w.r0 + r);
  }
}

// ---- the kernel on CUDA cores ------------------------------------------------
// 64 packed rows by tiles of 64 positions, 16 x 16 threads: thread (ty, tx)
// holds the scores of rows 4 ty.. and positions 4 tx.., and of its rows'
// outputs the dimensions 4 tx + 64 j. Everything float32.
constexpr int kCR = 64, kCT = 64, kCN = 256, kCS = 68;  // rows, tile, threads, padded row of the transposed tiles

template <int T, int HD>
__global__ void __launch_bounds__(kCN, 2) attn_chunk_kernel(const __grid_constant__ ChunkArgs a) {
  extern __shared__ __align__(16) float sm[];
  float *qs = sm;                  // [HD][kCS]: q transposed
  float *ks = qs + HD * kCS;       // [HD][kCS]: k transposed; then [kCT][kCS]: p transposed
  float *vs = ks + HD * kCS;       // [kCT][HD]
  __shared__ Plan plan;
  __shared__ long long warp_sums[kCN / 32];
  __shared__ long long prow[kCT];
  __shared__ unsigned arrived;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, hd = a.c.head_dim;
  static_assert(HD >= kCT, "the probabilities take the keys' place");
  make_plan<kCR, kCT, kCN>(a, &plan, warp_sums);
  Walk<kCR, kCT> w;
  w.start(a, plan);
  while (w.next(a)) {
    // queries, zeros past the unit's rows and past head_dim
    for (int i = tid; i < kCR * (HD / 4); i += kCN) {
      const int r = i % kCR, d = i / kCR * 4;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < w.nr && d < hd) {
        const int pr = w.r0 + r;
        ld4<T>(a.q, (long long)(w.s.q0 + pr / a.G) * a.ldq + (long long)(w.head * a.G + pr % a.G) * hd + d, v);
      }
#pragma unroll
      for (int e = 0; e < 4; e++) qs[(d + e) * kCS + r] = v[e];
    }
    int lim[4];
    float m[4], l[4], o[4][HD / 16];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      lim[r] = 4 * ty + r < w.nr ? visible(w.s, a.G, w.r0 + 4 * ty + r) : 0;
      m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
      for (int d = 0; d < HD / 16; d++) o[r][d] = 0.f;
    }
    for (int t = w.t0; t < w.t1; t++) {
      if (tid < kCT) prow[tid] = pool_row(a, w.s, w.b, w.head, t * kCT + tid);
      __syncthreads();
      for (int i = tid; i < kCT * (HD / 4); i += kCN) {
        const int p = i % kCT, d = i / kCT * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        const long long at = prow[p];
        if (at >= 0 && d < hd) ld4<T>(a.c.k_pool, at + d, v);
#pragma unroll
        for (int e = 0; e < 4; e++) ks[(d + e) * kCS + p] = v[e];
      }
      for (int i = tid; i < kCT * (HD / 4); i += kCN) {
        const int p = i / (HD / 4), d = i % (HD / 4) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        const long long at = prow[p];
        if (at >= 0 && d < hd) ld4<T>(a.c.v_pool, at + d, v);
        *(float4 *)(vs + p * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
      }
      __syncthreads();
      float s[4][4] = {};
#pragma unroll 8
      for (int d = 0; d < HD; d++) {
        const float4 q4 = *(const float4 *)(qs + d * kCS + 4 * ty), k4 = *(const float4 *)(ks + d * kCS + 4 * tx);
        const float qv[4] = {q4.x, q4.y, q4.z, q4.w}, kv[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int c = 0; c < 4; c++) s[r][c] = fmaf(qv[r], kv[c], s[r][c]);
      }
      __syncthreads();  // the keys are used up
#pragma unroll
      for (int r = 0; r < 4; r++) {
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          s[r][c] = t * kCT + 4 * tx + c < lim[r] ? s[r][c] * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, s[r][c]);
        }
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        const float mn = fmaxf(m[r], mx), ms = mn == -INFINITY ? 0.f : mn;
        const float f = ex2(m[r] - ms);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          s[r][c] = ex2(s[r][c] - ms);
          sum += s[r][c];
        }
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        l[r] = fmaf(l[r], f, sum);
        m[r] = mn;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) o[r][d] *= f;
      }
#pragma unroll
      for (int c = 0; c < 4; c++)
        *(float4 *)(ks + (4 * tx + c) * kCS + 4 * ty) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
      __syncthreads();
#pragma unroll 4
      for (int p = 0; p < kCT; p++) {
        const float4 p4 = *(const float4 *)(ks + p * kCS + 4 * ty);
        const float pv[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
        for (int j = 0; j < HD / 64; j++) {
          const float4 v4 = *(const float4 *)(vs + p * HD + 64 * j + 4 * tx);
#pragma unroll
          for (int r = 0; r < 4; r++) {
            o[r][4 * j] = fmaf(pv[r], v4.x, o[r][4 * j]);
            o[r][4 * j + 1] = fmaf(pv[r], v4.y, o[r][4 * j + 1]);
            o[r][4 * j + 2] = fmaf(pv[r], v4.z, o[r][4 * j + 2]);
            o[r][4 * j + 3] = fmaf(pv[r], v4.w, o[r][4 * j + 3]);
          }
        }
      }
      __syncthreads();  // the tile is used up
    }
    if (w.t0 == 0 && w.t1 == w.nt) {
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int pr = w.r0 + 4 * ty + r;
        const bool on = 4 * ty + r < w.nr;
        const float inv = l[r] > 0.f ? 1.f / l[r] : 0.f;
        const long long at = (long long)(w.s.q0 + pr / a.G) * a.ldo + (long long)(w.head * a.G + pr % a.G) * hd;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < HD / 64; j++)
          if (on && 64 * j + 4 * tx < hd) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = o[r][4 * j + k] * inv, odd |= !isfinite(v[k]);
            put4<T>(a.out, at + 64 * j + 4 * tx, v[0], v[1], v[2], v[3]);
          }
        const unsigned any = __ballot_sync(0xffffffffu, odd);
#pragma unroll
        for (int half = 0; half < 2; half++)
          if (any >> (16 * half) & 0xFFFFu)
            redo_row<T>(a, w.s, w.b, w.head, w.r0 + 4 * ((tid >> 5) * 2 + half) + r);
      }
      continue;
    }
    float *dst = part_slot<kCR>(a, blockIdx.x, w.t0 == 0);
#pragma unroll
    for (int r = 0; r < 4; r++) {
      if (4 * ty + r >= w.nr) continue;
#pragma unroll
      for (int j = 0; j < HD / 64; j++)
        *(float4 *)(dst + (size_t)(4 * ty + r) * kMaxHD + 64 * j + 4 * tx) =
            make_float4(o[r][4 * j], o[r][4 * j + 1], o[r][4 * j + 2], o[r][4 * j + 3]);
      if (tx == 0) {
        dst[kCR * kMaxHD + 4 * ty + r] = m[r];
        dst[kCR * (kMaxHD + 1) + 4 * ty + r] = l[r];
      }
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) arrived = atomicAdd(a.counter + w.c_first, 1u);
    __syncthreads();
    if (arrived != (unsigned)(w.c_last - w.c_first)) continue;
    __threadfence();
    join_pieces<T, kCR>(a, w, tid >> 5, kCN / 32);
    if (tid == 0) a.counter[w.c_first] = 0u;  // ready for the next launch
  }
}

template <int T, int HD>
int launch_simple(const ChunkArgs &a, int ctas, cudaStream_t st, const char *what) {
  const int smem = (2 * HD * kCS + kCT * HD) * (int)sizeof(float);
  GB_CUDA(cudaFuncSetAttribute(attn_chunk_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), what);
  attn_chunk_kernel<T, HD><<<(unsigned)ctas, kCN, smem, st>>>(a);
  GB_CUDA(cudaGetLastError(), what);
  return GB_OK;
}

}  // namespace

// Floats of partial rows and number of counters of a launch on `sms` SMs (two CTAs an SM).
size_t gb_attn_chunk_part_floats(int sms) { return (size_t)sms * 2 * 2 * kCR * (kMaxHD + 2); }
int gb_attn_chunk_counters(int sms) { return 2 * sms; }

int gb_attn_chunk_check(const gb_paged_chunk *c, const void *q, long long ldq, int n_heads, float scale,
                        const void *out, long long ldo) {
  const char *what = "gpu: chunk attention";
  const int rc = gb_paged_chunk_check(what, c);
  if (rc != GB_OK) return rc;
  const int hd = c->head_dim;
  if (hd < 16 || hd > kMaxHD || hd % 16)
    return gb_fail(GB_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 16 up to %d)", what, hd, kMaxHD);
  if (n_heads <= 0 || n_heads % c->n_kv)
    return gb_fail(GB_ERR_INVALID, "%s: %d heads is not a multiple of %d KV heads", what, n_heads, c->n_kv);
  // packed rows (row, query head of a group) are counted in 32 bits
  if (n_heads > (1 << 16) || (long long)c->rows * (n_heads / c->n_kv) > (1LL << 30))
    return gb_fail(GB_ERR_UNSUPPORTED, "%s: %d rows of %d heads", what, c->rows, n_heads);
  if (!(scale > 0.f) || isinf(scale)) return gb_fail(GB_ERR_INVALID, "%s: scale %g", what, scale);
  if (!q || !out || (((uintptr_t)q | (uintptr_t)out) & 15))
    return gb_fail(GB_ERR_INVALID, "%s: q or out is null or not on a 16-byte boundary", what);
  const long long wide = (long long)n_heads * hd;
  if (ldq % 8 || ldo % 8 || (c->rows > 1 && (ldq < wide || ldo < wide)))
    return gb_fail(GB_ERR_INVALID, "%s: rows %lld and %lld elements apart (multiples of 8, at least %lld)", what, ldq,
                   ldo, wide);
  return GB_OK;
}

int gb_attn_chunk_launch(const gb_paged_chunk *c, const void *q, long long ldq, int n_heads, float scale, void *out,
                         long long ldo, float *part, unsigned *counter, int sms, cudaStream_t st) {
  const char *what = "gpu: chunk attention";
  ChunkArgs a = {};
  a.c = *c;
  a.q = q, a.out = out, a.ldq = ldq, a.ldo = ldo;
  a.n_heads = n_heads, a.G = n_heads / c->n_kv;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.part = part, a.counter = counter;
#define GB_CHUNK(T) \
  if (c->kv_typ == T) return c->head_dim <= 64 ? launch_simple<T, 64>(a, 2 * sms, st, what) : launch_simple<T, 128>(a, 2 * sms, st, what);
  GB_CHUNK(GB_F32)
  GB_CHUNK(GB_F16)
  GB_CHUNK(GB_BF16)
#undef GB_CHUNK
  return gb_fail(GB_ERR_UNSUPPORTED, "%s: pool type %d", what, c->kv_typ);
}
