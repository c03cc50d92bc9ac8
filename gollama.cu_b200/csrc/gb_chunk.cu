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
// output) in the workspace, where they are joined in CTA order once all are
// there, so the result does not depend on which CTA does it. One rule
// serves one sequence decoding (a line of few units cut 148 ways), long
// prompts (whole units, cut only at the ends) and mixtures of both.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>

#include "gb_device.cuh"
#include "gb_internal.h"

namespace {

constexpr int kCounters = 3;
struct ChunkArgs {
  gb_paged_chunk c;
  const void *q;
  void *out;
  long long ldq, ldo;
  int n_heads, G;
  int q_tokens;       // of a TMA box of queries (0: none)
  float scale_log2;   // scale * log2(e): the softmax is taken in powers of two
  float *part;        // partial rows (part_slot)
  unsigned *counter;  // [CTAs][kCounters], zero between launches
  unsigned *err;      // a wait ran out (host memory)
  unsigned polls;     // of a barrier, before a wait runs out
};

// ---- the line of work --------------------------------------------------------

// A sequence as the device data describe it, made safe: rows outside the
// call's, or a table shorter than kv_len, cannot lead outside the buffers. Its
// rows stand where the append puts them, at kv_len - q_start[b + 1] + row, also
// where the call's rows end before the sequence's.
struct Seq {
  int q0, n;      // first row, new rows
  int len0;       // position of the first row (may be negative: rows that see nothing)
  int cap;        // positions the sequence holds, at most what its table can name
};
GB_DEV Seq seq_of(const ChunkArgs &a, int b) {
  Seq s;
  const int lo = max(0, a.c.q_start[b]), end = a.c.q_start[b + 1], hi = min(a.c.rows, max(lo, end));
  const int len = a.c.kv_lens[b];
  s.q0 = lo;
  s.n = max(0, hi - lo);
  s.len0 = s.n ? (int)max((long long)len - end + lo, -(1LL << 30)) : 0;  // n <= 2^30: none of them sees anything from there
  s.cap = min(max(len, 0), a.c.max_pages * a.c.page_size);
  return s;
}
// Positions that packed row r sees.
GB_DEV int visible(const Seq &s, int G, int r) { return max(0, min(s.cap, s.len0 + r / G + 1)); }

// The line is measured in costs, so that equal runs take equal times: a tile of
// a unit of more than RU / 2 rows costs WIDE, of a smaller one NARROW, and a
// unit's first tile OPEN more (its queries, the first tiles' latency, its
// rows' way out). A tile lies where it begins.
template <int RU, int KT, int WIDE, int NARROW, int OPEN>
struct Line {
  static GB_DEV int units(const Seq &s, int G) { return (int)(((long long)s.n * G + RU - 1) / RU); }
  // Tiles of unit u: up to the last position its last row sees; one where none is seen, so that the rows are written.
  static GB_DEV int tiles(const Seq &s, int G, int u) {
    const int last = (int)min((long long)s.n * G, (long long)(u + 1) * RU) - 1;
    return max(1, (visible(s, G, last) + KT - 1) / KT);
  }
  static GB_DEV int tile_cost(const Seq &s, int G, int u) {
    return (long long)s.n * G - (long long)u * RU > RU / 2 ? WIDE : NARROW;
  }
  static GB_DEV int cost(const Seq &s, int G, int u) { return OPEN + tiles(s, G, u) * tile_cost(s, G, u); }
  // Costs of the sequences of this warp's lanes, over all KV heads (no rows: none). A sequence of many units is
  // counted by the whole warp.
  static GB_DEV long long seq_cost(const ChunkArgs &a, const Seq &s) {
    const int lane = threadIdx.x & 31, nu = units(s, a.G);
    long long t = 0;
    if (nu <= 4)
      for (int u = 0; u < nu; u++) t += cost(s, a.G, u);
    for (unsigned many = __ballot_sync(0xffffffffu, nu > 4); many; many &= many - 1) {
      const int from = __ffs(many) - 1;
      Seq o;
      o.q0 = 0, o.n = __shfl_sync(0xffffffffu, s.n, from), o.len0 = __shfl_sync(0xffffffffu, s.len0, from);
      o.cap = __shfl_sync(0xffffffffu, s.cap, from);
      const int no = units(o, a.G);
      long long sum = 0;
      for (int u = lane; u < no; u += 32) sum += cost(o, a.G, u);
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
      if (lane == from) t = sum;
    }
    return t * a.c.n_kv;
  }
};

// x * y / z, in 32 bits where x * y fits.
GB_DEV long long mul_div(long long x, int y, long long z) {
  const unsigned long long p = (unsigned long long)x * (unsigned)y;
  if (p <= 0xFFFFFFFFull && z <= 0xFFFFFFFFll) return (uint32_t)p / (uint32_t)z;
  return (long long)(p / (unsigned long long)z);
}

struct Plan {
  long long total;   // the line's length
  long long x0, x1;  // this CTA's run of it: the tiles that begin there
  long long rem;     // x0's place within its sequence
  int ctas;          // the CTAs the line is cut for
  int b;             // the sequence x0 lies in
};
struct PlanShared {
  long long rem, warp_sums[32];
  int b;
};

GB_DEV long long warp_scan(long long v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// This CTA's run of a line of `total` whose tiles cost at most `most`. A run is
// no shorter than that, so that no CTA amid a unit is without a piece of it.
GB_DEV void cut_line(Plan &p, int most) {
  p.ctas = (int)min((long long)gridDim.x, (p.total + most - 1) / most);
  while (p.ctas > 1 && p.total < (long long)p.ctas * most) p.ctas--;
  const int me = min((int)blockIdx.x, p.ctas);
  p.x0 = p.ctas ? mul_div(p.total, me, p.ctas) : 0;
  p.x1 = me < p.ctas ? mul_div(p.total, me + 1, p.ctas) : p.x0;
}

// Every CTA finds its run by itself (a kernel of its own for it would cost a
// launch): the tiles of all sequences are counted and their sums scanned. Up to
// 64 sequences each warp does it alone, with no wait for the others; more are
// counted by the NT threads of the block together. All of them call it.
template <int RU, int KT, int WIDE, int NARROW, int OPEN, int NT>
GB_DEV Plan make_plan(const ChunkArgs &a, PlanShared *sp) {
  using L = Line<RU, KT, WIDE, NARROW, OPEN>;
  const int tid = threadIdx.x, lane = tid & 31, batch = a.c.batch;
  const Seq none = {0, 0, 0, 0};
  Plan p = {0, 0, 0, 0, 0, 0};
  if (batch <= 64) {
    const Seq q0 = lane < batch ? seq_of(a, lane) : none, q1 = lane + 32 < batch ? seq_of(a, lane + 32) : none;
    const bool wide = __any_sync(0xffffffffu, (long long)max(q0.n, q1.n) * a.G > RU / 2);
    const long long v0 = L::seq_cost(a, q0), v1 = batch > 32 ? L::seq_cost(a, q1) : 0;
    const long long s0 = warp_scan(v0), n0 = __shfl_sync(0xffffffffu, s0, 31), s1 = warp_scan(v1) + n0;
    p.total = __shfl_sync(0xffffffffu, s1, 31);
    cut_line(p, (wide ? WIDE : NARROW) + OPEN);
    const unsigned in0 = __ballot_sync(0xffffffffu, s0 - v0 <= p.x0 && p.x0 < s0);
    const unsigned in1 = __ballot_sync(0xffffffffu, s1 - v1 <= p.x0 && p.x0 < s1);
    const int at = in0 ? __ffs(in0) - 1 : in1 ? __ffs(in1) - 1 : 0;
    p.b = in0 ? at : at + 32;
    p.rem = p.x0 - __shfl_sync(0xffffffffu, in0 ? s0 - v0 : s1 - v1, at);
    return p;
  }
  // scans of NT sequences at a time: once for the total, once to find x0
  for (int pass = 0; pass < 2; pass++) {
    long long base = 0;
    for (int b0 = 0; b0 < batch; b0 += NT) {
      const long long v = L::seq_cost(a, b0 + tid < batch ? seq_of(a, b0 + tid) : none);
      long long s = warp_scan(v), sum = 0;
      __syncthreads();
      if (lane == 31) sp->warp_sums[tid >> 5] = s;
      __syncthreads();
      for (int w = 0; w < NT / 32; w++) {
        if (w == tid >> 5) s += sum;
        sum += sp->warp_sums[w];
      }
      if (pass && base + s - v <= p.x0 && p.x0 < base + s) {
        sp->b = b0 + tid;
        sp->rem = p.x0 - (base + s - v);
      }
      base += sum;
    }
    if (!pass) {
      p.total = base;
      cut_line(p, WIDE + OPEN);
    }
  }
  __syncthreads();
  p.b = sp->b, p.rem = sp->rem;
  return p;
}

// A walk over the pieces of this CTA's run: a piece is a unit's tiles [t0, t1).
template <int RU, int KT, int WIDE, int NARROW, int OPEN>
struct Walk {
  using L = Line<RU, KT, WIDE, NARROW, OPEN>;
  long long y, x1;  // where the unit begins; the run's end
  int b, u, h, i;   // sequence, unit, KV head, next tile
  // the piece
  Seq s;
  int r0, nr;      // the unit's packed rows [r0, r0 + nr) of the sequence
  int head;        // its KV head
  int t0, t1, nt;  // tiles of the piece, and of the unit
  int cost;        // of a tile

  // The first tile that begins at `pos` or later (from the unit's beginning).
  GB_DEV int tile_at(long long pos) const { return pos <= 0 ? 0 : pos <= OPEN ? 1 : (int)mul_div(pos - OPEN + cost - 1, 1, cost); }

  // All lanes of the warp call it: they look through the sequence's units 32 at a time.
  GB_DEV void start(const ChunkArgs &a, const Plan &p) {
    y = p.x0, x1 = p.x1;
    if (y >= x1) return;
    b = p.b;
    s = seq_of(a, b);
    long long rem = p.rem;
    const int lane = threadIdx.x & 31, nu = L::units(s, a.G);
    for (u = 0;; u += 32) {
      const int mine = u + lane < nu ? L::cost(s, a.G, u + lane) : 0;
      const long long sum = warp_scan((long long)mine * a.c.n_kv);  // with the units before it
      const unsigned past = __ballot_sync(0xffffffffu, sum > rem);
      if (past || u + 32 >= nu) {
        const int at = past ? __ffs(past) - 1 : 0;
        u += at;
        const int c = __shfl_sync(0xffffffffu, mine, at);
        rem -= __shfl_sync(0xffffffffu, sum, at) - (long long)c * a.c.n_kv;
        h = (int)mul_div(rem, 1, c);
        rem -= (long long)h * c;
        break;
      }
      rem -= __shfl_sync(0xffffffffu, sum, 31);
    }
    y -= rem;
    nt = L::tiles(s, a.G, u);
    cost = L::tile_cost(s, a.G, u);
    i = tile_at(rem);
    if (i >= nt) leave();
  }
  GB_DEV void leave() {
    y += OPEN + (long long)nt * cost;
    h++;
    i = 0;
  }
  GB_DEV bool next(const ChunkArgs &a) {
    if (y >= x1) return false;
    if (h == a.c.n_kv) {
      h = 0;
      if (++u == L::units(s, a.G)) {
        u = 0;
        do s = seq_of(a, ++b);
        while (s.n == 0);  // y < x1 <= total: a sequence with rows follows
      }
      nt = L::tiles(s, a.G, u);
      cost = L::tile_cost(s, a.G, u);
    }
    r0 = u * RU;
    nr = (int)min((long long)RU, (long long)s.n * a.G - r0);
    head = h;
    t0 = i;
    t1 = min(nt, tile_at(x1 - y));
    leave();
    return true;
  }
  // The CTAs that hold pieces of the unit just returned.
  GB_DEV void holders(const Plan &p, int *first, int *last) const {
    const long long y0 = y - OPEN - (long long)nt * cost, y1 = y0 + (nt > 1 ? OPEN + (nt - 1) * (long long)cost : 0);
    *first = (int)mul_div((y0 + 1) * p.ctas - 1, 1, p.total);
    *last = (int)mul_div((y1 + 1) * p.ctas - 1, 1, p.total);
  }
};

// The pool row of position p for KV head h, in units of `width` to a row, -1 past the
// sequence's positions; a table entry outside the pool reads page 0, as the
// decode attention does.
GB_DEV long long pool_row(const ChunkArgs &a, const Seq &s, int b, int h, int p, int width) {
  if (p >= s.cap) return -1;
  int phys = a.c.block_table[(long long)b * a.c.max_pages + p / a.c.page_size];
  if (phys < 0 || phys >= a.c.n_pages) phys = 0;
  return (((long long)phys * a.c.n_kv + h) * a.c.page_size + p % a.c.page_size) * width;
}

// ---- partial rows ------------------------------------------------------------
// A CTA leaves at most two pieces for others to join: the one its run begins
// within (which = 0) and the one it begins and does not end (which = 1). Each
// place holds kMaxHD floats of RU rows, four
// dimensions of all rows after another (a warp's rows store 512 bytes at a
// time), then what the rows' powers of two are taken from (their maxima, or
// near them) and their sums, kUnseen where a row sees no position of the
// piece: what lies there of its output is nothing of the row's, and is left
// out. A piece is not left out for a weight of zero, which does not stop a NaN
// in V that the row sees, wherever the line is cut.
constexpr float kUnseen = -1.f;
constexpr int kMaxHD = 128, kPlaces = 2;
template <int RU>
GB_DEV float *part_slot(const ChunkArgs &a, int cta, int which) {
  return a.part + (size_t)(cta * kPlaces + which) * RU * (kMaxHD + 2);
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
GB_DEV uint32_t pack2(float x, float y) {
  if constexpr (T == GB_F16) {
    const __half2 h = __floats2half2_rn(x, y);
    return *(const uint32_t *)&h;
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *(const uint32_t *)&h;
  }
}

// Eight results at an element index that is a multiple of 8.
template <int T>
GB_DEV void put8(void *out, long long i, const float *v) {
  if constexpr (T == GB_F32) {
    *(float4 *)((float *)out + i) = make_float4(v[0], v[1], v[2], v[3]);
    *(float4 *)((float *)out + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *(uint4 *)((uint16_t *)out + i) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}

// Four elements of type T from their 16 or 8 bytes.
template <int T>
GB_DEV void four(const uint4 &u, float *o) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if constexpr (T == GB_F32) o[e] = __uint_as_float(w[e]);
    else if constexpr (T == GB_F16) o[e] = gb_half_to_float((uint16_t)(w[e / 2] >> 16 * (e & 1)));
    else o[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
  }
}
template <int T>
GB_DEV void ld4(const void *base, long long i, float *o) {
  if constexpr (T == GB_F32) {
    four<T>(__ldg((const uint4 *)((const float *)base + i)), o);
  } else {
    const uint2 u = __ldg((const uint2 *)((const uint16_t *)base + i));
    four<T>(make_uint4(u.x, u.y, 0, 0), o);
  }
}

// ---- rows done again -----------------------------------------------------------
// A tile holds positions that some of its rows do not see, and their weight of
// zero does not stop a NaN or an infinity in V. So a row that came out with an
// infinity or NaN is looked at again, by one warp, and where they may be those of
// others done again by itself.
struct Unit {
  Seq s;
  int b, head, r0, nr, c_first, c_last;
};

// A lane's four elements (zeros past head_dim) of the pool row at `at`, -1: zeros.
template <int T>
GB_DEV void lane4(const void *pool, long long at, int hd, float *v) {
  const int lane = threadIdx.x & 31;
  const bool there = at >= 0 && 4 * lane < hd;
  ld4<T>(pool, there ? at + 4 * lane : 0, v);
  for (int e = 0; e < 4; e++) v[e] = there ? v[e] : 0.f;
}

// The last position with an infinity or NaN in V among those that the unit's
// tiles of KT hold and its first row does not see, -1: none.
template <int T, int KT>
GB_DEV int last_odd(const ChunkArgs &a, const Unit &w) {
  const int lane = threadIdx.x & 31, hd = a.c.head_dim, first = visible(w.s, a.G, w.r0);
  const int end = min(w.s.cap, max(1, (visible(w.s, a.G, w.r0 + w.nr - 1) + KT - 1) / KT) * KT);
  for (int p0 = end; p0 > first; p0 -= 32) {  // p0 - 1 and down
    const long long at = p0 - 1 - lane >= first ? pool_row(a, w.s, w.b, w.head, p0 - 1 - lane, hd) : -1;
    unsigned odd = 0;
#pragma unroll 8
    for (int j = 0; j < 32; j++) {
      float v[4];
      lane4<T>(a.c.v_pool, __shfl_sync(0xffffffffu, at, j), hd, v);
      if (!isfinite(v[0]) || !isfinite(v[1]) || !isfinite(v[2]) || !isfinite(v[3])) odd |= 1u << j;
    }
    odd = __reduce_or_sync(0xffffffffu, odd);
    if (odd) return p0 - __ffs(odd);
  }
  return -1;
}

// Whether each NaN of a row's results (this lane's four: r) has to be one: the row
// sees a NaN in K, or in V at that dimension.
template <int T>
GB_DEV bool sees_nan(const ChunkArgs &a, const Unit &w, int lim, float *r) {
  const int lane = threadIdx.x & 31, hd = a.c.head_dim;
  if (__any_sync(0xffffffffu, isinf(r[0]) || isinf(r[1]) || isinf(r[2]) || isinf(r[3]))) return false;
  for (int p0 = 0; p0 < lim; p0 += 32) {
    const long long at = p0 + lane < lim ? pool_row(a, w.s, w.b, w.head, p0 + lane, hd) : -1;
    bool nan = false;
#pragma unroll 4
    for (int j = 0; j < 32; j++) {
      const long long pj = __shfl_sync(0xffffffffu, at, j);
      float v[4], k[4];
      lane4<T>(a.c.v_pool, pj, hd, v);
      lane4<T>(a.c.k_pool, pj, hd, k);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (isnan(v[e])) r[e] = 0.f;
        nan = nan || isnan(k[e]);
      }
    }
    if (__any_sync(0xffffffffu, nan)) return true;
    if (!__any_sync(0xffffffffu, isnan(r[0]) || isnan(r[1]) || isnan(r[2]) || isnan(r[3]))) return true;
  }
  return false;
}

// A row by itself: lane = position for the scores, then lane = four dimensions
// for the sum over V, of which it writes those of the mask's bits (lane =
// position still, where that is one). It meets nothing but its own positions, so
// what it shows is its own: the NaN of 0 / 0 too, where every score it sees is
// -infinity.
template <int T>
GB_DEV void redo_row(const ChunkArgs &a, const Unit &w, int pr, int lim, unsigned mask) {
  const int lane = threadIdx.x & 31, hd = a.c.head_dim;
  const long long row = w.s.q0 + pr / a.G, hq = (long long)(w.head * a.G + pr % a.G) * hd;
  const int c4 = __popc(mask) == 1 ? __ffs(mask) - 1 : -1, my4 = c4 < 0 ? lane : c4;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < lim; p0 += 32) {
    const int p = p0 + lane;
    const long long at = p < lim ? pool_row(a, w.s, w.b, w.head, p, hd) : -1;
    float sc = 0.f;
    if (at >= 0)
#pragma unroll 8
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
    const int n = c4 < 0 ? min(32, lim - p0) : 1;
#pragma unroll 8
    for (int j = 0; j < n; j++) {
      const int from = c4 < 0 ? j : lane;
      const float pj = __shfl_sync(0xffffffffu, e, from);
      const long long vj = __shfl_sync(0xffffffffu, at, from);
      const bool there = 4 * my4 < hd && vj >= 0;
      float v[4];
      ld4<T>(a.c.v_pool, there ? vj + 4 * my4 : 0, v);
      for (int k = 0; k < 4; k++) o[k] = there ? fmaf(pj, v[k], o[k]) : o[k];
    }
  }
  if (c4 >= 0)
    for (int k = 0; k < 4; k++) o[k] = gb_warp_sum(o[k]);
  const float inv = lim > 0 ? 1.f / l : 0.f;
  if (4 * my4 < hd && (c4 < 0 ? mask >> lane & 1 : lane == 0))
    put4<T>(a.out, row * a.ldo + hq + 4 * my4, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}

// Looks at a unit's rows [lo, hi), `warps` warps in turn. What came out stands
// where the unit's tiles hold no infinity or NaN in V that the row does not see (a
// weight of zero was all that could go wrong; scores that it does not see are
// replaced), unless its weights had two parts, as an infinity times the remainder
// may be NaN, and where it has to be NaN in any case: all rows of a prompt done
// again for one NaN early in its V took 1,900 times a call's 95 us, and looked
// at like this take 1.7 times.
template <int T, int KT>
__device__ __noinline__ void redo_rows(const ChunkArgs &a, const Unit w, int lo, int hi, int warp, int warps) {
  const int lane = threadIdx.x & 31, hd = a.c.head_dim;
  const bool parts = T != GB_F32 && w.nr <= 128;
  int last = -2;  // not looked for
  for (int r = lo + warp; r < hi; r += warps) {
    const int pr = w.r0 + r, lim = visible(w.s, a.G, pr);
    const long long at = (long long)(w.s.q0 + pr / a.G) * a.ldo + (long long)(w.head * a.G + pr % a.G) * hd;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (4 * lane < hd) {
      if constexpr (T == GB_F32) {
        four<T>(__ldcg((const uint4 *)((const float *)a.out + at + 4 * lane)), v);
      } else {
        const uint2 x = __ldcg((const uint2 *)((const uint16_t *)a.out + at + 4 * lane));
        four<T>(make_uint4(x.x, x.y, 0, 0), v);
      }
    }
    const unsigned mask =
        __ballot_sync(0xffffffffu, !isfinite(v[0]) || !isfinite(v[1]) || !isfinite(v[2]) || !isfinite(v[3]));
    if (!mask) continue;
    if (last == -2) last = last_odd<T, KT>(a, w);
    if ((parts || last >= lim) && !sees_nan<T>(a, w, lim, v)) redo_row<T>(a, w, pr, lim, mask);
  }
}

GB_DEV void cp_async16(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Joins the pieces of a unit's rows [lo, hi), CTA by CTA, all NT threads of
// barrier 1 calling, with `room` bytes of shared memory to work in. First each row's weight of
// each piece, 2^(m_i - max) over the joined sum, several lanes to a row; then
// the rows, a thread to every so many runs of eight dimensions, whose pieces
// come through shared memory by asynchronous copies, as many of them on their
// way as fit: a unit of 256 rows brings 128 KB a piece, and with loads into
// registers each few of them cost a round trip to L2. `odd` is set where a result
// is an infinity or NaN: the caller looks at those rows, its own warps in step.
template <int T, int RU, int NT>
__device__ __noinline__ void join_pieces(const ChunkArgs &a, const Unit w, int tid, uint8_t *smem, int room, int lo,
                                         int hi, int *odd) {
  constexpr uint32_t kPlace = RU * (kMaxHD + 2), kStep = kPlaces * kPlace;  // floats of a place, of a CTA's places
  // in registers: through the reference each use is a load of some 200 clocks
  const float *const part = a.part + (uint32_t)w.c_first * kStep;  // piece i at i * kStep, the first in its second place
  void *const out = a.out;
  const int hd = a.c.head_dim, G = a.G, n = w.c_last - w.c_first + 1;
  if (hi - lo <= NT / 32) {  // few rows, often of many pieces: a warp to a row, a lane to four dimensions
    const int r = lo + (tid >> 5), lane = tid & 31, pr = w.r0 + r;
    if (r >= hi) return;
    bool any = false;  // the row sees a piece
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < n; i0 += 32) {
      float mi = -INFINITY, l_i = kUnseen;
      const int i = i0 + lane;
      if (i < n) {
        const float *p = part + ((uint32_t)i * kStep + (i ? 0 : kPlace) + RU * kMaxHD + r);
        mi = __ldcg(p), l_i = __ldcg(p + RU);
      }
      const unsigned seen = __ballot_sync(0xffffffffu, l_i != kUnseen);
      any = any || seen;
      if (l_i == kUnseen) l_i = 0.f;
      const float mn = fmaxf(m, gb_warp_max(mi)), ms = mn == -INFINITY ? 0.f : mn, g = ex2(m - ms), e = ex2(mi - ms);
      l = l * g + gb_warp_sum(e * l_i);
      o.x *= g, o.y *= g, o.z *= g, o.w *= g;
      m = mn;
      const float4 *p = (const float4 *)(part + ((uint32_t)i0 * kStep + (uint32_t)(min(lane, hd / 4 - 1) * RU + r) * 4));
      const int many = min(32, n - i0);
#pragma unroll 8
      for (int j = 0; j < many; j++) {
        const float4 v = __ldcg(p + (j * kStep + (i0 + j ? 0 : kPlace)) / 4);
        const float ej = __shfl_sync(0xffffffffu, e, j);
        if (seen >> j & 1) o.x = fmaf(ej, v.x, o.x), o.y = fmaf(ej, v.y, o.y), o.z = fmaf(ej, v.z, o.z), o.w = fmaf(ej, v.w, o.w);
      }
    }
    const float inv = any ? 1.f / l : 0.f;
    o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
    const bool fine = isfinite(o.x) && isfinite(o.y) && isfinite(o.z) && isfinite(o.w);
    if (4 * lane < hd)
      put4<T>(out, (long long)(w.s.q0 + pr / G) * a.ldo + (long long)(w.head * G + pr % G) * hd + 4 * lane, o.x, o.y, o.z, o.w);
    if (!fine) *(volatile int *)odd = 1;
    return;
  }
  float *const f = (float *)smem;  // [piece][row]
  // as many rows at a time as their weights take half the room at most
  const int most = max(1, min(hi - lo, room / 2 / (4 * n)));
  for (int r_lo = lo; r_lo < hi; r_lo += most) {
    const int nr = min(most, hi - r_lo);
    int log2_lanes = 0;  // lanes to a row
    while (log2_lanes < 5 && (2 << log2_lanes) * nr <= NT) log2_lanes++;
    const int lanes = 1 << log2_lanes, li = tid & (lanes - 1);
    for (int r0 = 0; r0 < nr; r0 += NT >> log2_lanes) {
      const int r = r0 + (tid >> log2_lanes);
      float m = -INFINITY, l = 0.f;
      if (r < nr)
#pragma unroll 4
        for (int i = li; i < n; i += lanes) {
          const float *p = part + ((uint32_t)i * kStep + (i ? 0 : kPlace) + RU * kMaxHD + r_lo + r);
          const float mi = __ldcg(p), l_i = __ldcg(p + RU), mn = fmaxf(m, mi), ms = mn == -INFINITY ? 0.f : mn;
          f[i * nr + r] = l_i == kUnseen ? NAN : mi;  // mi is none
          l = l * ex2(m - ms) + (l_i == kUnseen ? 0.f : l_i) * ex2(mi - ms);
          m = mn;
        }
      for (int o = 1; o < lanes; o <<= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m, o), lo = __shfl_xor_sync(0xffffffffu, l, o);
        const float mn = fmaxf(m, mo), ms = mn == -INFINITY ? 0.f : mn;
        l = l * ex2(m - ms) + lo * ex2(mo - ms);
        m = mn;
      }
      if (m == -INFINITY) m = 0.f;
      const float inv = 1.f / l;  // of a row that sees none, not used
      if (r < nr)
        for (int i = li; i < n; i += lanes) {
          const float mi = f[i * nr + r];
          f[i * nr + r] = isnan(mi) ? kUnseen : ex2(mi - m) * inv;
        }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
    const int table = (n * nr * 4 + 15) & ~15, pairs = (room - table) / (32 * NT);  // 32-byte pieces a thread holds
    float4 *const stage = (float4 *)(smem + table) + tid;  // slots 2 k and 2 k + 1: stage[2 k * NT], + NT
    const uint32_t stage_at = gb_smem_u32(stage);
    const int some = min(n, pairs), each = some == n ? pairs / some : 1;  // pieces, and runs of dimensions, at a time
    const int per = NT / nr, sub = tid / nr, r = tid - sub * nr, pr = w.r0 + r_lo + r, n8 = sub < per ? hd / 8 : 0;
    const int token = pr / G;
    const long long at = (long long)(w.s.q0 + token) * a.ldo + (long long)(w.head * G + pr - token * G) * hd;
    for (int q0 = sub; q0 < n8; q0 += each * per) {
      const int runs = min(each, (n8 - q0 + per - 1) / per);
      auto fetch = [&](int c8, int p0, uint32_t to) {  // pieces p0.. of a run
        const float *p = part + ((uint32_t)p0 * kStep + (uint32_t)(2 * c8 * RU + r_lo + r) * 4);
        const int many = min(some, n - p0);
#pragma unroll 4
        for (int i = 0; i < many; i++, p += kStep, to += 32 * NT) {
          const float *from = p + (p0 + i ? 0 : kPlace);
          cp_async16(to, from, true);
          cp_async16(to + 16 * NT, from + RU * 4, true);
        }
      };
      for (int k = 0; k < runs; k++) fetch(q0 + k * per, 0, stage_at + (uint32_t)(k * some) * 32 * NT);
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (int k = 0; k < runs; k++) {
        const int c8 = q0 + k * per;
        float o[8] = {};
        for (int p0 = 0; p0 < n; p0 += some) {
          if (p0) {  // more pieces than fit: the next ones
            fetch(c8, p0, stage_at);
            asm volatile("cp.async.wait_all;" ::: "memory");
          }
          const float *g = f + p0 * nr + r;
          const float4 *v = stage + (size_t)(k * some) * 2 * NT;
          const int many = min(some, n - p0);
#pragma unroll 4
          for (int i = 0; i < many; i++, g += nr, v += 2 * NT) {
            const float4 x = v[0], y = v[NT];
            const float gi = *g;
            if (gi != kUnseen) {
              o[0] = fmaf(gi, x.x, o[0]), o[1] = fmaf(gi, x.y, o[1]), o[2] = fmaf(gi, x.z, o[2]), o[3] = fmaf(gi, x.w, o[3]);
              o[4] = fmaf(gi, y.x, o[4]), o[5] = fmaf(gi, y.y, o[5]), o[6] = fmaf(gi, y.z, o[6]), o[7] = fmaf(gi, y.w, o[7]);
            }
          }
        }
        put8<T>(out, at + 8 * c8, o);
        bool fine = true;
#pragma unroll
        for (int e = 0; e < 8; e++) fine = fine && isfinite(o[e]);
        if (!fine) *(volatile int *)odd = 1;
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");  // the room is used up
  }
}

// ---- the kernel on CUDA cores (float32 pools) --------------------------------
// Up to ROWS packed rows by tiles of TILE positions, 16 x 16 threads, everything
// float32: thread (ty, tx) has the scores of rows ty + 16 i and positions tx +
// 16 j, and of its rows' outputs the dimensions 4 tx + 64 j. Both products read
// four elements at a time along their sum, so keys, values and queries stay in
// shared memory as they lie in the pools: a unit's i go up to NI = 1, 2, 4 or 8
// by its rows, and at 8 twelve 16-byte reads feed 128 multiply-adds. K of the
// next tile is on its way during the softmax and P V, V of it during Q K.
// 279 rows of 32 heads of 64 in two sequences of 1511 and 2048 positions: 148 us,
// 25.8 TFLOP/s; the multiply-add pipe is active 46 % of the time, the rest waits
// for shared memory and at dispatch.
constexpr int kFN = 256;  // threads
template <int HD>
struct F32 {
  static constexpr int ROWS = HD == 64 ? 128 : 64, TILE = HD == 64 ? 64 : 32;
  static constexpr int kRow = HD + 4, kP = TILE + 4;  // padded rows of Q and K, of P
  static constexpr int kFloats = ROWS * kRow + TILE * kRow + TILE * HD + ROWS * kP;
};

template <int HD>
__global__ void __launch_bounds__(kFN, 2) attn_chunk_f32_kernel(const __grid_constant__ ChunkArgs a) {
  using F = F32<HD>;
  constexpr int ROWS = F::ROWS, TILE = F::TILE, kRow = F::kRow, kP = F::kP, CJ = TILE / 16;
  extern __shared__ __align__(16) float sm[];
  float *const qs = sm, *const ks = qs + ROWS * kRow, *const vs = ks + TILE * kRow, *const ps = vs + TILE * HD;
  __shared__ PlanShared plan_shared;
  __shared__ Plan plan;
  __shared__ long long prow[2][TILE];
  __shared__ unsigned arrived;
  __shared__ int odd[2];  // an infinity or NaN in a row of a whole unit, of a joined one
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, hd = a.c.head_dim;
  Walk<ROWS, TILE, 1, 1, 0> w;
  {
    const Plan p = make_plan<ROWS, TILE, 1, 1, 0, kFN>(a, &plan_shared);
    w.start(a, p);
    if (tid == 0) plan = p, odd[0] = odd[1] = 0;
  }
  // a tile's rows to shared memory, `row` floats apart; zeros where there is none and past head_dim
  auto fetch = [&](const void *pool, int t, float *to, int row) {
    for (int i = tid; i < TILE * (HD / 4); i += kFN) {
      const int p = i / (HD / 4), d = i % (HD / 4) * 4;
      const long long at = prow[t & 1][p];
      const bool there = at >= 0 && d < hd;
      cp_async16(gb_smem_u32(to + p * row + d), (const float *)pool + (there ? at + d : 0), there);
    }
  };
  auto commit = []() { asm volatile("cp.async.commit_group;" ::: "memory"); };
  auto landed = []() { asm volatile("cp.async.wait_group 1;" ::: "memory"); };  // all but the last group
  auto unit = [&](auto ni) {
    constexpr int NI = decltype(ni)::value;
    if (tid < TILE) prow[w.t0 & 1][tid] = pool_row(a, w.s, w.b, w.head, w.t0 * TILE + tid, hd);
    for (int i = tid; i < 16 * NI * (HD / 4); i += kFN) {
      const int r = i / (HD / 4), d = i % (HD / 4) * 4, pr = w.r0 + r;
      const bool there = r < w.nr && d < hd;
      const long long at = (long long)(w.s.q0 + pr / a.G) * a.ldq + (long long)(w.head * a.G + pr % a.G) * hd + d;
      cp_async16(gb_smem_u32(qs + r * kRow + d), (const float *)a.q + (there ? at : 0), there);
    }
    __syncthreads();
    fetch(a.c.k_pool, w.t0, ks, kRow);
    commit();
    fetch(a.c.v_pool, w.t0, vs, HD);
    commit();
    const int all_see = visible(w.s, a.G, w.r0);  // positions that every row sees
    float m[NI], l[NI], o[NI][HD / 16];
#pragma unroll
    for (int i = 0; i < NI; i++) {
      m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
      for (int d = 0; d < HD / 16; d++) o[i][d] = 0.f;
    }
    for (int t = w.t0; t < w.t1; t++) {
      const bool more = t + 1 < w.t1;
      if (more && tid < TILE) prow[t + 1 & 1][tid] = pool_row(a, w.s, w.b, w.head, (t + 1) * TILE + tid, hd);
      landed();  // Q, K
      __syncthreads();
      float s[NI][CJ] = {};
#pragma unroll 2
      for (int d = 0; d < HD; d += 4) {
        float4 k4[CJ];
#pragma unroll
        for (int j = 0; j < CJ; j++) k4[j] = *(const float4 *)(ks + (tx + 16 * j) * kRow + d);
#pragma unroll
        for (int i = 0; i < NI; i++) {
          const float4 q4 = *(const float4 *)(qs + (ty + 16 * i) * kRow + d);
#pragma unroll
          for (int j = 0; j < CJ; j++)
            s[i][j] = fmaf(q4.x, k4[j].x, fmaf(q4.y, k4[j].y, fmaf(q4.z, k4[j].z, fmaf(q4.w, k4[j].w, s[i][j]))));
        }
      }
      __syncthreads();  // the keys are used up
      if (more) fetch(a.c.k_pool, t + 1, ks, kRow);
      commit();
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int lim = (t + 1) * TILE <= all_see ? all_see : visible(w.s, a.G, w.r0 + ty + 16 * i);
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < CJ; j++) {
          s[i][j] = t * TILE + tx + 16 * j < lim ? s[i][j] * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, s[i][j]);
        }
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.f : mn;
        const float f = ex2(m[i] - ms);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < CJ; j++) {
          s[i][j] = ex2(s[i][j] - ms);
          sum += s[i][j];
          ps[(ty + 16 * i) * kP + tx + 16 * j] = s[i][j];
        }
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        l[i] = fmaf(l[i], f, sum);
        m[i] = mn;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) o[i][d] *= f;
      }
      landed();  // V
      __syncthreads();
#pragma unroll 2
      for (int p = 0; p < TILE; p += 4) {
        float4 p4[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) p4[i] = *(const float4 *)(ps + (ty + 16 * i) * kP + p);
#pragma unroll
        for (int j = 0; j < HD / 64; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float4 v4 = *(const float4 *)(vs + (p + e) * HD + 64 * j + 4 * tx);
#pragma unroll
            for (int i = 0; i < NI; i++) {
              const float pe = e == 0 ? p4[i].x : e == 1 ? p4[i].y : e == 2 ? p4[i].z : p4[i].w;
              o[i][4 * j] = fmaf(pe, v4.x, o[i][4 * j]);
              o[i][4 * j + 1] = fmaf(pe, v4.y, o[i][4 * j + 1]);
              o[i][4 * j + 2] = fmaf(pe, v4.z, o[i][4 * j + 2]);
              o[i][4 * j + 3] = fmaf(pe, v4.w, o[i][4 * j + 3]);
            }
          }
      }
      __syncthreads();  // the values and weights are used up
      if (more) fetch(a.c.v_pool, t + 1, vs, HD);
      commit();
    }
    const bool whole = w.t0 == 0 && w.t1 == w.nt;
    float *const dst = part_slot<ROWS>(a, blockIdx.x, w.t0 == 0);
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int r = ty + 16 * i, pr = w.r0 + r;
      const bool on = r < w.nr;
      if (whole) {
        const float inv = visible(w.s, a.G, pr) > 0 ? 1.f / l[i] : 0.f;
        const long long at = (long long)(w.s.q0 + pr / a.G) * a.ldo + (long long)(w.head * a.G + pr % a.G) * hd;
        bool fine = true;
#pragma unroll
        for (int j = 0; j < HD / 64; j++)
          if (on && 64 * j + 4 * tx < hd) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = o[i][4 * j + k] * inv, fine = fine && isfinite(v[k]);
            put4<GB_F32>(a.out, at + 64 * j + 4 * tx, v[0], v[1], v[2], v[3]);
          }
        if (!fine) *(volatile int *)&odd[0] = 1;
      } else if (on) {
#pragma unroll
        for (int j = 0; j < HD / 64; j++)
          *(float4 *)(dst + ((16 * j + tx) * ROWS + r) * 4) =
              make_float4(o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]);
        if (tx == 0) {
          dst[ROWS * kMaxHD + r] = m[i];
          dst[ROWS * (kMaxHD + 1) + r] = visible(w.s, a.G, pr) > w.t0 * TILE ? l[i] : kUnseen;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // the empty groups
  };
  while (w.next(a)) {
    if (w.nr <= 16) unit(std::integral_constant<int, 1>());
    else if (w.nr <= 32) unit(std::integral_constant<int, 2>());
    else if (w.nr <= 64 || ROWS == 64) unit(std::integral_constant<int, 4>());
    else unit(std::integral_constant<int, ROWS / 16>());
    if (w.t0 == 0 && w.t1 == w.nt) continue;
    int c_first, c_last;
    w.holders(plan, &c_first, &c_last);
    __threadfence();
    __syncthreads();
    if (tid == 0) arrived = atomicAdd(a.counter + kCounters * c_first, 1u);
    __syncthreads();
    if (arrived != (unsigned)(c_last - c_first)) continue;
    __threadfence();
    const Unit u = {w.s, w.b, w.head, w.r0, w.nr, c_first, c_last};
    join_pieces<GB_F32, ROWS, kFN>(a, u, tid, (uint8_t *)sm, F::kFloats * (int)sizeof(float), 0, w.nr, &odd[1]);
    __syncthreads();
    if (odd[1]) redo_rows<GB_F32, TILE>(a, u, 0, w.nr, tid >> 5, kFN / 32);
    if (tid == 0) a.counter[kCounters * c_first] = 0u;  // ready for the next launch
  }
  __syncthreads();
  if (!odd[0]) return;
  w.start(a, plan);
  while (w.next(a))
    if (w.t0 == 0 && w.t1 == w.nt)
      redo_rows<GB_F32, TILE>(a, {w.s, w.b, w.head, w.r0, w.nr, 0, 0}, 0, w.nr, tid >> 5, kFN / 32);
}

// ---- the kernel on tensor cores (16-bit pools) --------------------------------
// Units of 256 packed rows, tiles of 128 positions. Both products run on
// tcgen05 (M = 128, float32 accumulators in tensor memory): S = Q K^T from
// shared memory, then O += P V with P written over S in tensor memory.
//
// Two softmax groups of eight warps; a row belongs to two threads, each with
// half of a tile's columns (and of O's): with a row to a thread a group took
// 3,000 clocks between scores and P, three times what the tensor cores take
// for its products, and there are too few warps to fill that. In a unit of more than
// 128 rows each group has 128 rows of its own and both use every tile; in a
// smaller one (decoding) both have the same rows and take alternate tiles, and
// their two results are joined like the pieces of two CTAs. Either way one
// group's softmax runs while the tensor cores work for the other.
//
// K and V tiles come in order K0 V0 K1 V1 ... into a ring, with the 128-byte
// swizzle that the descriptors name. Where the page size has a divisor of at
// least 8 in common with the tile, one warp fetches K and one V by TMA, in boxes
// of that many rows from wherever their page lies; what a box brings behind
// the sequence's end is overwritten with zeros in V (0 NaN is NaN) by a third
// warp, which also brings the queries, and does not matter in K. Other page
// sizes go through 16-byte asynchronous copies by the three warps, zeros behind
// the end. One thread issues all tcgen05.mma; they
// run in the order issued, so S of the next tile may be queued behind the P V
// that reads P in the same columns.
//
// The running maximum is let lag: the sums and outputs are rescaled only when
// a tile's maximum exceeds it by more than 2^kSlack, so most tiles leave O in
// tensor memory alone. In binary16, whose numbers end at 2^-24, the reference
// that a row's powers are taken from lies 2^kLift below the maximum (the sums
// and outputs have the same factor, and their quotient has none): P stays below
// 2^15 of the 65504 that the type holds, and a weight vanishes below 2^-32 of
// the row's largest, not below 2^-25, where many positions beside one that
// outweighs them would have lost up to 2^-25 each, all to the same side. A
// position adds 2^-32 at most to the error so.
//
// The tensor cores take P in 16 bits. A unit of more than 128 rows rounds it
// to the pool's type, as its result is rounded. Smaller units, which the
// cache's bytes bound, have room for P in two parts, the rounded one and the
// rounding's remainder (two products with V, in S's columns), and so none of
// that error but the numbers' end: few rows over few outstanding positions do
// not average it out.
//
// Measured in graphs: 64 sequences decoding at 1,200 to 8,000 positions (32
// heads over 8, head_dim 128) 214 us, 5.6 TB/s of the cache's bytes, in bursts of
// 13 ms at 1.97 GHz, and 237 to 247 where the power limit holds the clock at 1.5;
// 2048 rows of 64 heads behind 14,336 positions 1.01 ms, 1.02 PFLOP/s, under that limit. What bounds long chunks is the exchange between a
// group's softmax and the products: of a tile's 4,000 clocks the tensor cores
// work 2,000, and with neither exponentials nor products 2,900 remain.
constexpr int kTR = 256, kTT = 128;       // rows of a unit, positions of a tile
constexpr int kSoftWarps = 16, kLoadWarps = 3, kMmaWarp = kSoftWarps + kLoadWarps;
constexpr int kTN = (kMmaWarp + 1) * 32;  // threads
constexpr float kSlack = 8.f;
template <int T>
constexpr float kLift = T == GB_F16 ? 7.f : 0.f;
constexpr int kSlice = 64, kPolls = 64;  // rows joined at a time; polls (some 0.8 us) for a unit's other holders
constexpr uint32_t kChunkBytes = 128 * 128;  // 128 rows of 64 elements
constexpr int kRingBytes = 10 * kChunkBytes;
template <int HD>
constexpr int ring_slots() { return kRingBytes / (HD / 64 * (int)kChunkBytes); }
constexpr int kHeader = 3 * 1024;  // tiles lie on 1024-byte boundaries behind it
template <int HD>
constexpr int tc_smem() { return kHeader + 2 * HD / 64 * (int)kChunkBytes + kRingBytes; }

struct TcShared {
  uint64_t full[10], empty[10], landed[10], q_full, q_empty, s_full[2], p_full[2][2], pv_done[2], o_free, fin;
  PlanShared plan;
  Plan mine;  // this CTA's, for its end
  uint32_t tmem;
  int dead, odd[2];      // a wait ran out; an infinity or NaN in a row of a whole unit, of a joined one
  uint32_t fetched[2];   // ring places up to which K and V were fetched
  Unit unit[2];          // the pieces left in this CTA's places (nr = 0: none)
  int slice[2], busy[2];  // the first row to join of each; whether to come again
  float top[2][2][128];  // what the two threads of a row tell each other
};
static_assert(sizeof(TcShared) <= kHeader, "shared header");

GB_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
GB_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
GB_DEV void tc_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(gb_smem_u32(bar))
               : "memory");
}
// D[128 x N] (+)= A B^T, both from shared memory.
GB_DEV void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same with A from tensor memory.
GB_DEV void tc_mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Columns of this warp's 32 lanes into registers. The wait is part of the same
// statement: the loads are asynchronous, and between them and a wait of its own
// the compiler may move the results, or give their registers to other values.
GB_DEV void tc_ld16(uint32_t addr, uint32_t *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16]; "
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}
GB_DEV void tc_ld32(uint32_t addr, uint32_t *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
      "%28,%29,%30,%31}, [%32]; "
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
        "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]),
        "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
GB_DEV void tc_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(
          r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
GB_DEV void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory descriptors, 128-byte swizzle, 128-byte rows in groups of
// eight (1024 bytes). Rows along M or N with K contiguous (Q, K): the groups
// are the stride. Rows along K with N contiguous (V): the groups are the
// stride along K, and 64-element column chunks (kChunkBytes) the leading one.
GB_DEV uint64_t desc_rows(uint32_t saddr, uint32_t leading) {
  const uint32_t lo = (saddr >> 4 & 0x3FFFu) | (leading >> 4 << 16);
  return (uint64_t)((1024u >> 4) | 1u << 14 | 2u << 29) << 32 | lo;
}
// Where P's 16 positions 16 k.. lie among S's columns: the 32 columns of
// scores 32 h.. hold their P (16 columns), then its remainder, so that no
// score is overwritten before it is read.
GB_DEV constexpr int p_column(int k) { return 32 * (k >> 1) + 8 * (k & 1); }
// kind::f16: float32 accumulators, A and B of type T, B with N contiguous when TB.
template <int T>
GB_DEV uint32_t idesc_of(int N, bool TB) {
  const uint32_t f = T == GB_BF16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (TB ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((128u >> 4) << 24);
}

// Every wait is bounded: when one runs out, or another thread's has, it returns
// false, `dead` is set and the error word tells. The CTA then ends by these
// rules (all addresses stay within their buffers):
// - a warp that fetches starts no copy once it sees `dead`. The products go on
//   and may report a slot empty that was never filled, but only with `dead` set
//   before, so no barrier that counts a copy's bytes is arrived at before that
//   copy has landed, and at most one copy of a slot is on its way;
// - the softmax warps go on without waiting: they meet at barriers of the block,
//   and the units' other holders count on this CTA's arrival;
// - the last waits (`last`: for copies and products in flight) are made all the
//   same.
// `tiles`: how many tiles' work the wait spans, of any length in a long sequence.
// `dead` is looked at each 64th poll: with each of them one sequence decoding took
// 28.1 us instead of 26.7, and a long chunk 1,060 instead of 1,030.
GB_DEV bool bar_wait(TcShared *sh, uint64_t *bar, uint32_t parity, const ChunkArgs &a, bool last = false, int tiles = 1) {
  const uint32_t polls = last ? GB_WAIT_LIMIT : a.polls;
  for (int t = 0; t < tiles; t++)
    for (uint32_t i = 0; i < polls; i++) {
      if (gb_mbar_try_wait(bar, parity)) return true;
      if (!last && (i & 63) == 63 && *(volatile int *)&sh->dead) return false;
    }
  *(volatile int *)&sh->dead = 1;
  *(volatile unsigned *)a.err = GB_DEVERR_TIMEOUT;
  return false;
}
// The same for a warp that fetches: whether it may go on.
GB_DEV bool fetch_wait(TcShared *sh, uint64_t *bar, uint32_t parity, const ChunkArgs &a, int tiles = 1) {
  return __all_sync(0xffffffffu, bar_wait(sh, bar, parity, a, false, tiles) && !*(volatile int *)&sh->dead);
}

GB_DEV void cp_async_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(gb_smem_u32(bar)) : "memory");
}

// A warp's copies of its 32 rows of a tile: `at` is the lane's row (elements
// from base, -1: zeros), ppr 16-byte pieces a row, several rows a pass.
template <int PPR>
GB_DEV void load_rows_of(const uint16_t *base, long long at, uint32_t tile, int row0, int ppr, int lane) {
  const int pr = PPR ? PPR : ppr, rpp = 32 / pr, sub = lane / pr, pc = lane - sub * pr;
  const uint32_t chunk = tile + (uint32_t)(pc >> 3) * kChunkBytes;
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += rpp) {
    const int r = r0 + sub;
    const long long from = __shfl_sync(0xffffffffu, at, r & 31);
    if (sub < rpp && r < 32) {
      const int row = row0 + r;
      cp_async16(chunk + row * 128 + ((pc ^ row) & 7) * 16, base + (from < 0 ? 0 : from) + pc * 8, from >= 0);
    }
  }
}
GB_DEV void load_rows(const uint16_t *base, long long at, uint32_t tile, int row0, int ppr, int lane) {
  if (ppr == 16) load_rows_of<16>(base, at, tile, row0, ppr, lane);  // unrolled: 40 clocks a pass otherwise
  else if (ppr == 8) load_rows_of<8>(base, at, tile, row0, ppr, lane);
  else load_rows_of<0>(base, at, tile, row0, ppr, lane);
}

// A unit's queries, 32 rows at a time in turn by `warps` warps; zeros past its
// rows, except that whole 32 rows past them are left as they are (no softmax
// warp looks at those).
GB_DEV void load_q(const ChunkArgs &a, const Seq &s, int u0, int nr, int head, uint32_t q_at, uint32_t tile, int lw,
                   int warps, int ppr, int lane) {
  for (int j = lw; j * 32 < nr; j += warps) {
    const int r = j * 32 + lane, pr = u0 + r;
    const long long at =
        r < nr ? (long long)(s.q0 + pr / a.G) * a.ldq + (long long)(head * a.G + pr % a.G) * a.c.head_dim : -1;
    load_rows((const uint16_t *)a.q, at, q_at + (j >> 2) * tile, (j & 3) * 32, ppr, lane);
  }
}

// The rows a TMA box holds: the page size's common divisor with a tile.
__host__ GB_DEV int box_rows(int page_size) {
  const int low = page_size & -page_size;
  return low < kTT ? low : kTT;
}

GB_DEV uint32_t elect_lane() {
  uint32_t on;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(on));
  return on;
}

GB_DEV void tma_box(uint32_t dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(gb_smem_u32(bar))
      : "memory");
}

GB_DEV void tma_box3(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(gb_smem_u32(bar))
      : "memory");
}

// What a packed pair leaves of (x, y): the remainder, exact in float32.
template <int T>
GB_DEV uint32_t pack2_rest(float x, float y, uint32_t p) {
  if constexpr (T == GB_F16) {
    const float2 f = __half22float2(*(const __half2 *)&p);
    return pack2<T>(x - f.x, y - f.y);
  } else {
    return pack2<T>(x - __uint_as_float(p << 16), y - __uint_as_float(p & 0xFFFF0000u));
  }
}

// Two float32 in one register pair.
GB_DEV uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
GB_DEV void unpair(uint64_t r, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r)); }
GB_DEV uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
GB_DEV uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
// P of this warp's rows from 64 columns of scores at s_at, in their place: powers
// of two of s * scale + shift, rounded to T (and the remainders, unless BOTH);
// the sum of a row's. With `cut`, columns from `rel` on are not seen. The exponential unit's four a clock and
// scheduler do not bound it: with a quarter of the powers formed by a polynomial
// on the multiply-add units it took as long. The loop stays rolled: straight code
// for a tile outgrows the schedulers' instruction caches, and fetching it took as
// long as running it (stalls on no instruction as many as issues).
template <int T, bool BOTH>
GB_DEV float weights(uint32_t s_at, int rel, bool cut, float scale, float shift, uint64_t *full) {
  const uint64_t k2 = pair(scale, scale), c2 = pair(shift, shift);
  uint64_t sum[2] = {0, 0};
#pragma unroll 1
  for (int h = 0; h < 2; h++) {
    uint32_t u[32], rest[16];
    tc_ld32(s_at + 32 * h, u);
    if (cut)
#pragma unroll
      for (int c = 0; c < 32; c++) u[c] = 32 * h + c < rel ? u[c] : 0xFF800000u;  // -infinity
#pragma unroll
    for (int c = 0; c < 16; c++) {
      float x, y;
      unpair(fma2(pair(__uint_as_float(u[2 * c]), __uint_as_float(u[2 * c + 1])), k2, c2), x, y);
      x = ex2(x), y = ex2(y);
      sum[c & 1] = add2(sum[c & 1], pair(x, y));
      u[c] = pack2<T>(x, y);
      if (!BOTH) rest[c] = pack2_rest<T>(x, y, u[c]);
    }
    tc_st16(s_at + 32 * h, u);
    if (!BOTH) tc_st16(s_at + 32 * h + 16, rest);
    tc_wait_st();
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) gb_mbar_arrive(full + h);
  }
  float x, y;
  unpair(add2(sum[0], sum[1]), x, y);
  return x + y;
}

template <int T, int HD, bool TMA>
__global__ void __launch_bounds__(kTN, 1)
    attn_chunk_tc_kernel(const __grid_constant__ ChunkArgs a, const __grid_constant__ CUtensorMap k_map,
                         const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap q_map) {
  extern __shared__ __align__(1024) uint8_t tc_raw[];
  TcShared *const sh = (TcShared *)tc_raw;
  const uint32_t q_at = gb_smem_u32(tc_raw) + kHeader;
  constexpr uint32_t kTile = HD / 64 * kChunkBytes;
  constexpr int NS = ring_slots<HD>();
  const uint32_t ring = q_at + 2 * kTile;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hd = a.c.head_dim;
  if (warp == 0) {
    if (lane < NS) {
      gb_mbar_init(&sh->full[lane], TMA ? 1 : kLoadWarps * 32);
      gb_mbar_init(&sh->empty[lane], 1);
      gb_mbar_init(&sh->landed[lane], 1);
    } else if (lane < NS + 2) {
      const int g = lane - NS;
      gb_mbar_init(&sh->s_full[g], 1);
      gb_mbar_init(&sh->p_full[g][0], kSoftWarps / 2);
      gb_mbar_init(&sh->p_full[g][1], kSoftWarps / 2);
      gb_mbar_init(&sh->pv_done[g], 1);
    } else if (lane == 31) {
      gb_mbar_init(&sh->q_full, (TMA ? 1 : kLoadWarps) * 32);
      gb_mbar_init(&sh->q_empty, 1);
      gb_mbar_init(&sh->o_free, kSoftWarps);
      gb_mbar_init(&sh->fin, 1);
      sh->dead = sh->odd[0] = sh->odd[1] = sh->unit[0].nr = sh->unit[1].nr = 0;
    }
    gb_mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(gb_smem_u32(&sh->tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // A wide tile takes 4,000 clocks, a narrow one 2,200, and what a piece has before and behind its tiles some 6,000
  // (counted as 4,000, 12 ragged sequences took 111 us instead of 105; as twice a tile of the unit's kind, 112). The
  // tiles were traced at head_dim 128 with TMA; the other forms are cut by the same costs.
  const Plan plan = make_plan<kTR, kTT, 4, 2, 6, kTN>(a, &sh->plan);
  Walk<kTR, kTT, 4, 2, 6> w;
  w.start(a, plan);
  if (tid == 0) sh->mine = plan;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;

  if (TMA && warp < kSoftWarps + 2 && warp >= kSoftWarps) {
    // ---- K (one warp) and V (another) by TMA: lane i finds box i's row, one lane
    // issues the boxes, a 64-element column chunk each (all lanes their own took
    // 130 clocks a box)
    const int kv = warp - kSoftWarps, br = box_rows(a.c.page_size), box = lane & (kTT / br - 1);
    constexpr int chunks = HD / 64;
    const uint32_t leader = elect_lane();
    const CUtensorMap *const map = kv ? &v_map : &k_map;
    uint32_t n = 0, ends = 0, phase = 0;  // bits of the slots: the last copy is a sequence's end; parity of the next landing
    bool live = true;
    while (live && w.next(a)) {
      const int32_t *const table = a.c.block_table + (long long)w.b * a.c.max_pages;
      int p = w.t0 * kTT + box * br, page = p / a.c.page_size;
      int phys = p < w.s.cap ? table[page] : 0;
      for (int t = w.t0; t < w.t1; t++, n += 2) {
        const int y0 = ((phys < 0 || phys >= a.c.n_pages ? 0 : phys) * a.c.n_kv + w.head) * a.c.page_size +
                       p - page * a.c.page_size;
        // the next tile's table entry is on its way while this one's rows are
        p += kTT;
        page = p / a.c.page_size;
        phys = t + 1 < w.t1 && p < w.s.cap ? table[page] : 0;
        const int held = min(max(w.s.cap - t * kTT, 0), kTT), boxes = (held + br - 1) / br;
        const uint32_t slot = (n + kv) % NS;
        live = fetch_wait(sh, &sh->empty[slot], ((n + kv) / NS & 1) ^ 1, a);
        if (!live) break;
        // V at the sequence's end goes through the warp that puts the zeros, which then reports it full
        const bool end = kv && held < kTT;
        uint64_t *bar = end ? &sh->landed[slot] : &sh->full[slot];
        ends = (ends & ~(1u << slot)) | (uint32_t)end << slot;
        phase ^= (uint32_t)end << slot;
        if (lane == 0) gb_mbar_expect_tx(bar, (uint32_t)(boxes * chunks * br) * 128);
        __syncwarp();
        for (int i = 0; i < boxes; i++) {
          const int y = __shfl_sync(0xffffffffu, y0, i);
          const uint32_t to = ring + slot * kTile + (uint32_t)(i * br) * 128;
          if (leader) {
            tma_box(to, map, 0, y, bar);
            if (HD > 64) tma_box(to + kChunkBytes, map, 64, y, bar);
          }
        }
        __syncwarp();
      }
    }
    // Whatever was fetched has landed before the CTA ends. What lies NS and more places before the last fetch has been
    // read; of the others a slot's last one is waited for, whichever warp it is (another fetch follows a read).
    if (lane == 0) sh->fetched[kv] = n;
    asm volatile("bar.sync 14, 64;" ::: "memory");
    for (uint32_t i = n > NS ? n - NS - 1 : 0; i < n; i++) {
      const uint32_t slot = i % NS;
      if ((i & 1) != (uint32_t)kv || i + NS < sh->fetched[(i + NS) & 1]) continue;
      if (ends >> slot & 1) bar_wait(sh, &sh->landed[slot], (phase >> slot & 1) ^ 1, a, true);
      else bar_wait(sh, &sh->full[slot], i / NS & 1, a, true);
    }
  } else if (TMA && warp == kSoftWarps + 2) {
    // ---- queries, and zeros over V behind the sequence's end
    const int ppr = hd / 8;
    const uint32_t leader = elect_lane();
    uint32_t n0 = 0, pieces = 0, phase = 0;  // bit i: parity of the next landing in slot i
    int before = 1;                          // tiles of the piece before
    while (w.next(a)) {
      if (!fetch_wait(sh, &sh->q_empty, (pieces & 1) ^ 1, a, before)) break;
      before = w.t1 - w.t0;
      // Where 128 packed rows are whole tokens' heads they are a box: 256 rows took this warp 4.4 us by
      // copies of its own. The box brings rows past the unit's too, which nobody looks at; few rows are copied.
      if (a.q_tokens && w.nr > 32) {
        const int halves = w.nr > 128 ? 2 : 1;
        if (lane == 0) gb_mbar_expect_tx(&sh->q_full, halves * kTile);
        else gb_mbar_arrive(&sh->q_full);
        __syncwarp();
        if (leader)
          for (int i = 0; i < halves; i++)
            for (int c = 0; c < HD / 64; c++)
              tma_box3(q_at + i * kTile + c * kChunkBytes, &q_map, 64 * c, w.head * a.G,
                       w.s.q0 + w.r0 / a.G + i * a.q_tokens, &sh->q_full);
        __syncwarp();
      } else {
        load_q(a, w.s, w.r0, w.nr, w.head, q_at, kTile, 0, 1, ppr, lane);
        cp_async_arrive(&sh->q_full);
      }
      pieces++;
      const int last = w.s.cap / kTT;  // the tile that the end lies in
      if (last >= w.t0 && last < w.t1) {
        const uint32_t slot = (n0 + 2 * (last - w.t0) + 1) % NS;
        if (!fetch_wait(sh, &sh->landed[slot], phase >> slot & 1, a, before)) break;
        phase ^= 1u << slot;
        for (int i = (w.s.cap % kTT) * 8 + lane; i < kTT * 8; i += 32)
          for (int c = 0; c < HD / 64; c++)
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring + slot * kTile + c * kChunkBytes + i * 16),
                         "r"(0)
                         : "memory");
        gb_fence_proxy_async();
        __syncwarp();
        if (lane == 0) gb_mbar_arrive(&sh->full[slot]);
      }
      n0 += 2 * (w.t1 - w.t0);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (pieces) bar_wait(sh, &sh->q_full, (pieces - 1) & 1, a, true);
  } else if (!TMA && warp >= kSoftWarps && warp < kMmaWarp) {
    // ---- queries, K and V by asynchronous copies
    // A tile's four blocks of 32 rows go round the three warps, one block on with each tile.
    const int lw = warp - kSoftWarps, ppr = hd / 8;
    uint32_t n = 0, pieces = 0;
    bool live = true;
    auto block = [&](int t, int k) { return (lw + 3 - t % 3) % 3 + 3 * k; };  // k = 0, 1; 4 and on: none
    auto row_of = [&](int t, int k) {
      const int j = block(t, k);
      return t < w.t1 && j < 4 ? pool_row(a, w.s, w.b, w.head, t * kTT + j * 32 + lane, hd) : -1;
    };
    while (live && w.next(a)) {
      live = fetch_wait(sh, &sh->q_empty, (pieces & 1) ^ 1, a);
      if (!live) break;
      load_q(a, w.s, w.r0, w.nr, w.head, q_at, kTile, lw, kLoadWarps, ppr, lane);
      cp_async_arrive(&sh->q_full);
      pieces++;
      long long at0 = row_of(w.t0, 0), at1 = row_of(w.t0, 1);
      for (int t = w.t0; live && t < w.t1; t++) {
        // the next tile's table entries are on their way while this one's rows are
        const long long ahead0 = row_of(t + 1, 0), ahead1 = row_of(t + 1, 1);
#pragma unroll
        for (int kv = 0; kv < 2; kv++, n++) {
          const uint32_t slot = n % NS;
          live = live && fetch_wait(sh, &sh->empty[slot], (n / NS & 1) ^ 1, a);
          if (!live) break;
          const uint16_t *pool = (const uint16_t *)(kv ? a.c.v_pool : a.c.k_pool);
          load_rows(pool, at0, ring + slot * kTile, block(t, 0) * 32, ppr, lane);
          if (block(t, 1) < 4) load_rows(pool, at1, ring + slot * kTile, block(t, 1) * 32, ppr, lane);
          cp_async_arrive(&sh->full[slot]);
        }
        at0 = ahead0, at1 = ahead1;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kMmaWarp) {
    // ---- the products: the warp walks and waits together, one elected lane issues
    // The lane's own predicate, as elect.sync gives it: with more put into it (a lane's number, whether a wait ran out)
    // the products were compiled with operands that were not the warp's.
    const uint32_t leader = elect_lane();
    const uint32_t iq = idesc_of<T>(kTT, false), iv = idesc_of<T>(hd, true);
    uint32_t n0 = 0, pieces = 0, np0 = 0, np1 = 0;  // ring position of the piece, pieces, P's taken of each group
    // S_g = Q_qt K^T, K at ring position n; `k_done`: its slot's last use; `q_done`: the queries' last use
    auto qk = [&](int g, int qt, uint32_t n, bool k_done, bool q_done) {
      const uint32_t k_at = ring + n % NS * kTile, x_at = q_at + qt * kTile;
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++) {
          const uint32_t off = (uint32_t)(kk >> 2) * kChunkBytes + (uint32_t)(kk & 3) * 32;
          if (16 * kk < hd) tc_mma(tmem + g * 128, desc_rows(x_at + off, 16), desc_rows(k_at + off, 16), iq, kk != 0);
        }
        tc_commit(&sh->s_full[g]);
        if (k_done) tc_commit(&sh->empty[n % NS]);
        if (q_done) tc_commit(&sh->q_empty);
      }
      __syncwarp();
    };
    // O_g (+)= P_g V, V at ring position n
    auto pv = [&](int g, uint32_t n, bool first, bool both, bool v_done) {
      const uint32_t v_at = ring + n % NS * kTile, parity = (g ? np1++ : np0++) & 1;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        bar_wait(sh, &sh->p_full[g][h], parity, a);
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int k = 0; k < kTT / 32; k++) {
            const int kk = 4 * (k >> 1) + 2 * h + (k & 1);
            tc_mma_ta(tmem + 256 + g * 128, tmem + g * 128 + p_column(kk), desc_rows(v_at + kk * 2048, kChunkBytes), iv,
                      !first || h || k);
            if (!both)
              tc_mma_ta(tmem + 256 + g * 128, tmem + g * 128 + p_column(kk) + 16,
                        desc_rows(v_at + kk * 2048, kChunkBytes), iv, 1);
          }
        }
        __syncwarp();
      }
      if (leader) {
        tc_commit(&sh->pv_done[g]);
        if (v_done) tc_commit(&sh->empty[n % NS]);
      }
      __syncwarp();
    };
    auto loaded = [&](uint32_t n) {
      bar_wait(sh, &sh->full[n % NS], n / NS & 1, a);
      // the asynchronous copies' bytes, seen here, before the tensor cores read them (about 400 cycles)
      if (!TMA) gb_fence_proxy_async();
    };
    while (w.next(a)) {
      const int n = w.t1 - w.t0;
      const bool both = w.nr > 128;  // both groups use each tile
      bar_wait(sh, &sh->q_full, pieces & 1, a);
      gb_fence_proxy_async();
      loaded(n0);
      if (both) {
        qk(0, 0, n0, false, false);
        qk(1, 1, n0, true, n == 1);
      } else {
        qk(0, 0, n0, true, n == 1);
        if (n > 1) {
          loaded(n0 + 2);
          qk(1, 0, n0 + 2, true, n == 2);
        }
      }
      bar_wait(sh, &sh->o_free, (pieces & 1) ^ 1, a);  // O of the last unit has been read
      for (int t = 0; t < n; t++) {
        const uint32_t v = n0 + 2 * t + 1;
        loaded(v);
        if (both) {
          if (t + 1 < n) loaded(v + 1);
          pv(0, v, t == 0, true, false);
          if (t + 1 < n) qk(0, 0, v + 1, false, false);
          pv(1, v, t == 0, true, true);
          if (t + 1 < n) qk(1, 1, v + 1, true, t + 2 == n);
        } else {
          const int g = t & 1;
          pv(g, v, t < 2, false, true);
          if (t + 2 < n) {
            loaded(v + 3);
            qk(g, 0, v + 3, true, t + 3 == n);
          }
        }
      }
      n0 += 2 * n;
      pieces++;
    }
    // nothing is in flight when the tensor memory is given back
    if (leader) tc_commit(&sh->fin);
    __syncwarp();
    bar_wait(sh, &sh->fin, 0, a, true);
  } else {
    // ---- softmax: two threads to a row
    const int g = warp >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21, s_at = tmem + g * 128 + 64 * half + lanes;
    float *const my_top = &sh->top[g][half][row], *const other_top = &sh->top[g][half ^ 1][row];
    const int pair_bar = 2 + g * 4 + (warp & 3);
    auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory"); };
    uint32_t ns = 0;  // tiles this group has taken
    while (w.next(a)) {
      const bool both = w.nr > 128;
      const int ur = (both ? g * 128 : 0) + row, pr = w.r0 + ur;
      const bool mine = ur < w.nr;
      const bool warp_on = ur - lane < w.nr;
      // rows past the unit's in a warp of its rows have zeros for queries, or by TMA other tokens', and are not looked at
      const int lim = mine ? visible(w.s, a.G, pr) : 0x7FFFFFFF;
      float m = -INFINITY, l = 0.f;
      int done = 0;
      for (int t = w.t0 + (both ? 0 : g); t < w.t1; t += both ? 1 : 2, ns++, done++) {
        bar_wait(sh, &sh->s_full[g], ns & 1, a);
        tc_fence_after();
        if (warp_on) {
          // the scores are read twice, once for the maximum and once for P: kept in
          // registers they spilled
          const int rel = lim - t * kTT - 64 * half;
          const bool cut = __any_sync(0xffffffffu, rel < 64);
          float top = -INFINITY;
#pragma unroll 1
          for (int h = 0; h < 2; h++) {
            uint32_t u[32];
            tc_ld32(s_at + 32 * h, u);
            if (cut)
#pragma unroll
              for (int c = 0; c < 32; c++) u[c] = 32 * h + c < rel ? u[c] : 0xFF800000u;  // -infinity
            float mx[4];
#pragma unroll
            for (int c = 0; c < 4; c++) mx[c] = __uint_as_float(u[c]);
#pragma unroll
            for (int c = 4; c < 32; c++) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(u[c]));
            top = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          }
          // both threads of a row go by the larger maximum
          *my_top = top;
          pair_sync();
          top = fmaxf(top, *other_top) * a.scale_log2;
          const bool raise = top > m + (kSlack + kLift<T>) || m == -INFINITY;
          const float mn = raise ? fmaxf(m, top - kLift<T>) : m;
          if (__any_sync(0xffffffffu, raise)) {
            const float f = mn == -INFINITY ? 1.f : ex2(m - mn);
            l *= f;
            if (done) {  // O is there: the last P V must have ended before it is scaled
              bar_wait(sh, &sh->pv_done[g], (ns - 1) & 1, a);
              tc_fence_after();
              for (int c = half; c < hd / 16; c += 2) {
                const uint32_t o_at = tmem + 256 + g * 128 + lanes + 16 * c;
                uint32_t u[16];
                tc_ld16(o_at, u);
#pragma unroll
                for (int e = 0; e < 16; e++) u[e] = __float_as_uint(__uint_as_float(u[e]) * f);
                tc_st16(o_at, u);
              }
            }
          }
          m = mn;
          const float ms = m == -INFINITY ? 0.f : m;
          l += both ? weights<T, true>(s_at, rel, cut, a.scale_log2, -ms, sh->p_full[g])
                    : weights<T, false>(s_at, rel, cut, a.scale_log2, -ms, sh->p_full[g]);
        } else if (lane < 2) {
          gb_mbar_arrive(&sh->p_full[g][lane]);
        }
      }
      // ---- the unit's end: its rows out of tensor memory. The threads of a row
      // (two, or four where both groups have it) tell each other their sums,
      // then their maxima, and take 16 columns of O in turn. Warps without rows
      // keep step: none reports O free twice before another has once.
      const bool whole = w.t0 == 0 && w.t1 == w.nt;
      if (done) {
        bar_wait(sh, &sh->pv_done[g], (ns - 1) & 1, a);
        tc_fence_after();
      }
      float f0 = 1.f, f1 = 0.f;  // weights of this group's result (both), or of the two groups'
      *my_top = l;
      if (both) {
        pair_sync();
        l += *other_top;
        pair_sync();  // read before it is written again
      } else {
        const int quad_bar = 10 + (warp & 3);
        auto quad_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(quad_bar) : "memory"); };
        tc_fence_before();  // both groups' products have ended
        quad_sync();
        tc_fence_after();
        const float l0 = sh->top[0][0][row] + sh->top[0][1][row], l1 = sh->top[1][0][row] + sh->top[1][1][row];
        quad_sync();
        *my_top = m;
        quad_sync();
        const float m0 = sh->top[0][0][row], m1 = sh->top[1][0][row];
        quad_sync();
        m = fmaxf(m0, m1);
        const float ms = m == -INFINITY ? 0.f : m;
        f0 = ex2(m0 - ms), f1 = ex2(m1 - ms);
        l = f0 * l0 + f1 * l1;
      }
      if (warp_on) {
        const bool two = !both && w.t1 - w.t0 > 1;  // group 1 has had a tile
        const float inv = !whole ? 1.f : lim > 0 ? 1.f / l : 0.f;
        f0 *= inv, f1 *= inv;
        bool odd = false;
        const long long at = (long long)(w.s.q0 + pr / a.G) * a.ldo + (long long)(w.head * a.G + pr % a.G) * hd;
        float *const dst = part_slot<kTR>(a, blockIdx.x, w.t0 == 0);
        const uint32_t o_at = tmem + 256 + (both ? g * 128 : 0) + lanes;
        for (int c = both ? half : 2 * g + half; c < hd / 16; c += both ? 2 : 4) {
          uint32_t u[16];
          float o[16];
          tc_ld16(o_at + 16 * c, u);
#pragma unroll
          for (int e = 0; e < 16; e++) o[e] = __uint_as_float(u[e]) * f0;
          if (two) {
            tc_ld16(o_at + 128 + 16 * c, u);
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = fmaf(__uint_as_float(u[e]), f1, o[e]);
          }
          if (!mine) continue;
          if (whole) {
#pragma unroll
            for (int e = 0; e < 16; e++) odd |= !isfinite(o[e]);
#pragma unroll
            for (int e = 0; e < 16; e += 8) put8<T>(a.out, at + 16 * c + e, o + e);
          } else {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *(float4 *)(dst + ((4 * c + e / 4) * kTR + ur) * 4) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (!whole && mine && !half && (both || !g)) {
          dst[kTR * kMaxHD + ur] = m;
          dst[kTR * (kMaxHD + 1) + ur] = lim > w.t0 * kTT ? l : kUnseen;
        }
        if (odd) *(volatile int *)&sh->odd[0] = 1;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) gb_mbar_arrive(&sh->o_free);
      if (!whole && tid == 0) {
        Unit u = {w.s, w.b, w.head, w.r0, w.nr, 0, 0};
        w.holders(sh->mine, &u.c_first, &u.c_last);
        sh->unit[w.t0 == 0] = u;
      }
    }
    // ---- the CTA's end: the joining of the units it has left pieces of, and rows
    // with an infinity or a NaN done again (calls within the loop above cost it
    // registers). The holders of a unit arrive at it; once all have, its rows are
    // taken in slices by whoever is there (one CTA alone took 10 us for 256
    // rows). Who comes early waits for the others, who end at about the same
    // time, but not long: the last to arrive is always there to do what is left.
    // The last to leave makes the unit's counters ready for the next launch.
    auto all = []() { asm volatile("bar.sync 1, %0;" ::"n"(kSoftWarps * 32) : "memory"); };
    __threadfence();
    all();
    const Unit *const my_unit = &sh->unit[tid & 1];  // of the first two threads
    unsigned *const counter = a.counter + kCounters * my_unit->c_first;
    const unsigned holders = (unsigned)(my_unit->c_last - my_unit->c_first + 1);
    bool there = false, busy = tid < 2 && my_unit->nr;
    if (busy) there = atomicAdd(counter, 1u) == holders - 1;
    for (;;) {
      if (tid < 2) {
        for (int k = 0; busy && !there && k < kPolls; k++) {
          there = *(volatile unsigned *)counter == holders;
          if (!there) __nanosleep(100);
        }
        const int lo = busy && there ? (int)atomicAdd(counter + 1, 1u) * kSlice : my_unit->nr;
        sh->slice[tid] = lo;
        busy = lo + kSlice < my_unit->nr;  // there may be another
        sh->busy[tid] = busy;
      }
      __threadfence();
      all();
      const int lo[2] = {sh->slice[0], sh->slice[1]};
      for (int i = 0; i < 2; i++) {
        const Unit &u = sh->unit[i];
        // in the tiles' room: all of them are used up
        if (lo[i] < u.nr)
          join_pieces<T, kTR, kSoftWarps * 32>(a, u, tid, tc_raw + kHeader, tc_smem<HD>() - kHeader, lo[i],
                                               min(lo[i] + kSlice, u.nr), &sh->odd[1]);
      }
      const bool more = sh->busy[0] || sh->busy[1];
      all();
      if (sh->odd[1] && !sh->dead)  // what comes of a wait that ran out is not looked at
        for (int i = 0; i < 2; i++) redo_rows<T, kTT>(a, sh->unit[i], lo[i], min(lo[i] + kSlice, sh->unit[i].nr), warp, kSoftWarps);
      if (!more) break;
    }
    if (tid < 2 && my_unit->nr && atomicAdd(counter + 2, 1u) == holders - 1) counter[0] = counter[1] = counter[2] = 0u;
    if (sh->odd[0] && !sh->dead) {
      w.start(a, sh->mine);
      while (w.next(a))
        if (w.t0 == 0 && w.t1 == w.nt)
          redo_rows<T, kTT>(a, {w.s, w.b, w.head, w.r0, w.nr, 0, 0}, 0, w.nr, warp, kSoftWarps);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// 16-bit elements in boxes whose rows are 64 of them, zeros past the dims.
int tensor_map(void *base, int rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
               CUtensorMap *map, const char *what) {
  static EncodeTiledFn encode = nullptr;
  if (!encode) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess || !fn)
      return gb_fail(GB_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", what);
    encode = (EncodeTiledFn)fn;
  }
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, rank, base, dims, strides, box, one,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return gb_fail(GB_ERR_CUDA, "%s: tensor map encode failed (%d)", what, (int)r);
  return GB_OK;
}

// A pool as rows of head_dim elements, in boxes of `br` rows.
int pool_map(const ChunkArgs &a, void *pool, int br, CUtensorMap *map, const char *what) {
  const cuuint64_t dims[2] = {(cuuint64_t)a.c.head_dim, (cuuint64_t)a.c.n_pages * a.c.n_kv * a.c.page_size};
  const cuuint64_t strides[1] = {(cuuint64_t)a.c.head_dim * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)br};
  return tensor_map(pool, 2, dims, strides, box, map, what);
}

// The queries [rows][n_heads][head_dim], in boxes of a KV head's G heads of 128 / G tokens.
int query_map(const ChunkArgs &a, CUtensorMap *map, const char *what) {
  const cuuint64_t dims[3] = {(cuuint64_t)a.c.head_dim, (cuuint64_t)a.n_heads, (cuuint64_t)a.c.rows};
  const cuuint64_t row = a.c.rows > 1 ? (cuuint64_t)a.ldq : (cuuint64_t)a.n_heads * a.c.head_dim;  // of one row: any
  const cuuint64_t strides[2] = {(cuuint64_t)a.c.head_dim * 2, row * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)a.G, (cuuint32_t)a.q_tokens};
  return tensor_map((void *)a.q, 3, dims, strides, box, map, what);
}

template <int T, int HD, bool TMA>
int launch_tc(ChunkArgs a, int sms, cudaStream_t st, const char *what) {
  CUtensorMap k_map = {}, v_map = {}, q_map = {};
  if (TMA) {
    const int br = box_rows(a.c.page_size);
    int rc = pool_map(a, a.c.k_pool, br, &k_map, what);
    if (rc == GB_OK) rc = pool_map(a, a.c.v_pool, br, &v_map, what);
    a.q_tokens = 128 % a.G ? 0 : 128 / a.G;
    if (rc == GB_OK && a.q_tokens) rc = query_map(a, &q_map, what);
    if (rc != GB_OK) return rc;
  }
  GB_CUDA(cudaFuncSetAttribute(attn_chunk_tc_kernel<T, HD, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               tc_smem<HD>()),
          what);
  attn_chunk_tc_kernel<T, HD, TMA><<<(unsigned)sms, kTN, tc_smem<HD>(), st>>>(a, k_map, v_map, q_map);
  GB_CUDA(cudaGetLastError(), what);
  return GB_OK;
}

template <int T>
int launch_16(const ChunkArgs &a, int sms, cudaStream_t st, const char *what) {
  // a box starts on a group of eight swizzled rows, and its row is a 32-bit coordinate
  const bool tma = box_rows(a.c.page_size) >= 8 && (long long)a.c.n_pages * a.c.n_kv * a.c.page_size < (1LL << 31);
  if (a.c.head_dim <= 64) return tma ? launch_tc<T, 64, true>(a, sms, st, what) : launch_tc<T, 64, false>(a, sms, st, what);
  return tma ? launch_tc<T, 128, true>(a, sms, st, what) : launch_tc<T, 128, false>(a, sms, st, what);
}

template <int HD>
int launch_f32(const ChunkArgs &a, int ctas, cudaStream_t st, const char *what) {
  constexpr int smem = F32<HD>::kFloats * (int)sizeof(float);
  GB_CUDA(cudaFuncSetAttribute(attn_chunk_f32_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), what);
  attn_chunk_f32_kernel<HD><<<(unsigned)ctas, kFN, smem, st>>>(a);
  GB_CUDA(cudaGetLastError(), what);
  return GB_OK;
}

}  // namespace

// Floats of partial rows and number of counters of a launch on `sms` SMs: two
// CTAs an SM in float32, one on the tensor cores.
size_t gb_attn_chunk_part_floats(int sms) {
  return (size_t)sms * kPlaces * std::max(2 * F32<64>::ROWS, kTR) * (kMaxHD + 2);
}
int gb_attn_chunk_counters(int sms) { return 2 * sms * kCounters; }

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
  if (!gb_paged_chunk_any(c)) return GB_OK;
  if (!q || !out || (((uintptr_t)q | (uintptr_t)out) & 15))
    return gb_fail(GB_ERR_INVALID, "%s: q or out is null or not on a 16-byte boundary", what);
  const long long wide = (long long)n_heads * hd;
  if (ldq % 8 || ldo % 8 || (c->rows > 1 && (ldq < wide || ldo < wide)))
    return gb_fail(GB_ERR_INVALID, "%s: rows %lld and %lld elements apart (multiples of 8, at least %lld)", what, ldq,
                   ldo, wide);
  return GB_OK;
}

int gb_attn_chunk_launch(const gb_paged_chunk *c, const void *q, long long ldq, int n_heads, float scale, void *out,
                         long long ldo, float *part, unsigned *counter, unsigned *err, unsigned polls, int sms,
                         cudaStream_t st) {
  const char *what = "gpu: chunk attention";
  ChunkArgs a = {};
  a.c = *c;
  a.q = q, a.out = out, a.ldq = ldq, a.ldo = ldo;
  a.n_heads = n_heads, a.G = n_heads / c->n_kv;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.part = part, a.counter = counter, a.err = err, a.polls = polls;
  if (c->kv_typ == GB_F32)
    return c->head_dim <= 64 ? launch_f32<64>(a, 2 * sms, st, what) : launch_f32<128>(a, 2 * sms, st, what);
  if (c->kv_typ == GB_F16) return launch_16<GB_F16>(a, sms, st, what);
  if (c->kv_typ == GB_BF16) return launch_16<GB_BF16>(a, sms, st, what);
  return gb_fail(GB_ERR_UNSUPPORTED, "%s: pool type %d", what, c->kv_typ);
}
