// gb_rows.cu -- per-head work on the rows a projection leaves behind: norms
// of queries and keys for each head, the position rotation (cpu.RoPE,
// backend/cpu/cpu.go:118-138), and the append of keys and values to a paged
// cache, each element read once and written once.
//
// For a head's row x of head_dim elements, in float32:
//   norm      x' = x * w / sqrt(mean(x^2) + eps)
//   rotation  the pair (a, b) at (2j, 2j+1), or (j, j + dims/2) in halves,
//             becomes (a cos t - b sin t, a sin t + b cos t) with
//             t = pos * base^(-2j/dims) / freq[j], j < dims/2.
// The angle is formed in float64 as a number of turns, t / (2 pi), whose
// fraction alone goes to sincospi: at position 2^20 a float32 angle would be
// off by 2^-4 radians, while the float64 turn is off by about 1e-11.
#include <math.h>

#include <algorithm>

#include <cuda_bf16.h>

#include "gb_device.cuh"
#include "gb_internal.h"

namespace {

constexpr int kMaxHD = 256;       // head_dim
constexpr int kMaxThreads = 192;  // threads of a CTA, a task each

struct RowArgs {
  const void *q, *k, *v;  // rows of n_heads / n_kv / n_kv heads (v only for the append)
  void *q_out, *k_out;    // k_out only without the append
  long long ldq, ldk, ldv, ldqo, ldko;  // elements between rows
  int nq, nk, nv;         // heads of q, k, v
  int hd, dims, halves;
  int lph_log2;           // lanes per head (16 elements a lane)
  const float *wq, *wk, *freq;
  float eps;
  double log2_step;       // of the angles' ratio: -2 log2(base) / dims
  const int32_t *pos;     // without the append
  int rows;
  gb_paged_chunk c;       // with the append
};

// Eight elements of type T: their bytes, and their values.
template <int T>
struct Raw {
  uint4 u[T == GB_F32 ? 2 : 1];
};
template <int T>
GB_DEV Raw<T> fetch8(const void *base, long long i) {
  Raw<T> r;
  if constexpr (T == GB_F32) {
    r.u[0] = *(const uint4 *)((const float *)base + i);
    r.u[1] = *(const uint4 *)((const float *)base + i + 4);
  } else {
    r.u[0] = *(const uint4 *)((const uint16_t *)base + i);
  }
  return r;
}
template <int T>
GB_DEV void values8(const Raw<T> &r, float *o) {
  const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if constexpr (T == GB_F32) {
      o[e] = __uint_as_float(w[e]);
    } else if constexpr (T == GB_F16) {
      o[2 * e] = gb_half_to_float((uint16_t)w[e]);
      o[2 * e + 1] = gb_half_to_float((uint16_t)(w[e] >> 16));
    } else {
      o[2 * e] = __uint_as_float(w[e] << 16);
      o[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
    }
  }
  if constexpr (T == GB_F32) {
    const uint32_t v[4] = {r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
#pragma unroll
    for (int e = 0; e < 4; e++) o[4 + e] = __uint_as_float(v[e]);
  }
}

template <int T>
GB_DEV void st8(void *base, long long i, const float *v) {
  if constexpr (T == GB_F32) {
    *(float4 *)((float *)base + i) = make_float4(v[0], v[1], v[2], v[3]);
    *(float4 *)((float *)base + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if constexpr (T == GB_F16) {
        const __half2 h = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
        w[e] = *(const uint32_t *)&h;
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
        w[e] = *(const uint32_t *)&h;
      }
    }
    *(uint4 *)((uint16_t *)base + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// One task: a lane's 16 elements of one head, as two runs of eight at dA and
// dB. In halves a run pairs with the other one, so no lane needs another
// lane's elements; side by side the pairs lie within a run.
struct Task {
  int head, dA, dB;
  bool on, rot;
};
GB_DEV Task task_of(const RowArgs &a, int t) {
  Task k;
  const int l = t & ((1 << a.lph_log2) - 1);
  k.head = t >> a.lph_log2;
  k.on = 16 * l < a.hd && k.head < a.nq + a.nk + a.nv;
  if (a.halves && 16 * l < a.dims) {
    k.dA = 8 * l, k.dB = 8 * l + a.dims / 2;
  } else {
    k.dA = 16 * l, k.dB = 16 * l + 8;
  }
  k.rot = 16 * l < a.dims && k.head < a.nq + a.nk;
  return k;
}

// Where a task's elements lie in row 0, and the distance between rows.
GB_DEV const void *task_source(const RowArgs &a, const Task &k, long long *at, long long *ld) {
  const int h = k.head < a.nq ? k.head : k.head < a.nq + a.nk ? k.head - a.nq : k.head - a.nq - a.nk;
  *at = (long long)h * a.hd;
  *ld = k.head < a.nq ? a.ldq : k.head < a.nq + a.nk ? a.ldk : a.ldv;
  return k.head < a.nq ? a.q : k.head < a.nq + a.nk ? a.k : a.v;
}

// Waits until at most n of this thread's groups of copies (n known when the loop
// over rows is unrolled) are on their way.
GB_DEV void rows_landed(int n) {
  if (n >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (n == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_all;" ::: "memory");
}

// R rows by a slice of their heads to a CTA, a thread to the same 16 elements of
// a head in each row: all rows' elements are on their way while the rows'
// sequences are looked up (by each warp for itself) and their R dims/2 angles
// formed, once for all heads. R is 1, or 4 by the rule of four_rows(), the
// elements then on their way to shared memory, where a thread reads what it
// asked for. With float32 rows, of which two fit, 8192 rows of 40 heads took 60
// us against 43, and the append of 8192 rows of 48 heads 33.5 against 31. CTAs of
// up to 192 threads: 320 took 66, 37, 47 and 31, 128 took 64, 40, 46 and 30.5.
// Few rows are bound by the launch: 2.3 us for one, 3 for 64 with their append
// (launches of one graph).
template <int TI, int TO, bool APPEND, int R>
__global__ void __launch_bounds__(kMaxThreads, R > 1 ? 5 : 1) head_rows_kernel(const __grid_constant__ RowArgs a) {
  static_assert(R == 1 || (sizeof(Raw<TI>) == 16 && !APPEND), "rows by way of shared memory");
  __shared__ float2 cs[R][kMaxHD / 2];          // pair j of row i at [i][(j % 8) * half / 8 + j / 8]
  extern __shared__ uint4 stage[];              // [row][run][thread]
  const int row0 = blockIdx.x * R, tid = threadIdx.x, lane = tid & 31, half = a.dims / 2, eighth = half / 8;
  const Task k = task_of(a, (int)(blockIdx.y * blockDim.x) + tid);
  Raw<TI> xa = {}, xb = {};
  long long src_at, ld;
  const void *const src = task_source(a, k, &src_at, &ld);
  if constexpr (R == 1) {
    if (k.on) {
      xa = fetch8<TI>(src, row0 * ld + src_at + k.dA);
      xb = fetch8<TI>(src, row0 * ld + src_at + k.dB);
    }
  } else {
    const uint32_t to = gb_smem_u32(stage + tid);
#pragma unroll
    for (int i = 0; i < R; i++) {
      if (k.on && row0 + i < a.rows) {
        const uint16_t *from = (const uint16_t *)src + (row0 + i) * ld + src_at;
#pragma unroll
        for (int run = 0; run < 2; run++)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (uint32_t)(2 * i + run) * blockDim.x * 16),
                       "l"(from + (run ? k.dB : k.dA))
                       : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  // lane i knows row i: whether it belongs to a sequence, its position, and the
  // element index of its slot in head 0 of its page (-1: none)
  const int row = row0 + lane;
  bool there = lane < R && row < a.rows;
  long long p = 0, slot = -1;
  if constexpr (APPEND) {  // one row: lane 0's
    int b = -1;
    for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
      const bool in = b0 + lane < a.c.batch;
      const int lo = in ? a.c.q_start[b0 + lane] : 0, hi = in ? a.c.q_start[b0 + lane + 1] : 0;
      const unsigned hit = __ballot_sync(0xffffffffu, lo <= row0 && row0 < hi);
      if (lane == 0 && b < 0 && hit) b = b0 + __ffs(hit) - 1;
      if (__all_sync(0xffffffffu, !there || b >= 0)) break;
    }
    there = there && b >= 0;
    if (there) {
      p = (long long)a.c.kv_lens[b] - a.c.q_start[b + 1] + row;
      if (p >= 0 && p < (long long)a.c.max_pages * a.c.page_size) {
        const int at = (int)p, n = at / a.c.page_size, page = a.c.block_table[(long long)b * a.c.max_pages + n];
        if (page >= 0 && page < a.c.n_pages)
          slot = ((long long)page * a.c.n_kv * a.c.page_size + at - n * a.c.page_size) * a.hd;
      }
    }
  } else if (there && a.pos) {
    p = a.pos[row];
  }
  const unsigned rows_there = __ballot_sync(0xffffffffu, there);
  for (int at0 = 0; at0 < R * half; at0 += blockDim.x) {
    const int at = at0 + tid, i = min(at / max(half, 1), R - 1), j = at - i * half;
    const long long pi = __shfl_sync(0xffffffffu, p, i);
    if (at < R * half) {
      double turns = (double)pi * exp2(a.log2_step * j) * 0.15915494309189535;  // 1 / (2 pi)
      if (a.freq) turns /= (double)a.freq[j];
      float2 &c = cs[i][(j & 7) * eighth + (j >> 3)];  // a warp's lanes read neighbours
      sincospif((float)(2.0 * (turns - rint(turns))), &c.y, &c.x);
    }
  }
  __syncthreads();
  const bool is_q = k.head < a.nq, is_v = k.head >= a.nq + a.nk;
  const float *w = is_q ? a.wq : is_v ? nullptr : a.wk;
  const int h = is_q ? k.head : k.head - a.nq - (is_v ? a.nk : 0);
  const int l8 = (a.halves ? k.dA : k.dA / 2) >> 3;  // the task's pairs are 8 l8 ..
#pragma unroll
  for (int i = 0; i < R; i++) {
    if constexpr (R > 1) {
      rows_landed(R - 1 - i);
      // lanes past head_dim asked for nothing and add nothing to their head's sum
      xa.u[0] = k.on ? stage[2 * i * blockDim.x + tid] : make_uint4(0, 0, 0, 0);
      xb.u[0] = k.on ? stage[(2 * i + 1) * blockDim.x + tid] : make_uint4(0, 0, 0, 0);
    }
    float x[16];
    values8<TI>(xa, x);
    values8<TI>(xb, x + 8);
    const long long slot_i = __shfl_sync(0xffffffffu, slot, i);
    if (a.wq || a.wk) {
      // the lanes of a head sit in one warp and agree on w, but a warp's heads may
      // differ: the sum is formed by all lanes, and used where there is a weight
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e++) ss = fmaf(x[e], x[e], ss);
      for (int o = 1; o < (1 << a.lph_log2); o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (k.on && w) {
        const float r = rsqrtf(ss / (float)a.hd + a.eps);
        float wv[8];
        values8<GB_F32>(fetch8<GB_F32>(w, k.dA), wv);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = x[e] * r * wv[e];
        values8<GB_F32>(fetch8<GB_F32>(w, k.dB), wv);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e + 8] = x[e + 8] * r * wv[e];
      }
    }
    if (!k.on || !(rows_there >> i & 1)) continue;
    if (k.rot) {
      if (R > 1 || a.halves) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float2 c = cs[i][e * eighth + l8];
          const float u = x[e], v = x[e + 8];
          x[e] = u * c.x - v * c.y;
          x[e + 8] = u * c.y + v * c.x;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float2 c = cs[i][e * eighth + l8];
          const float u = x[2 * e], v = x[2 * e + 1];
          x[2 * e] = u * c.x - v * c.y;
          x[2 * e + 1] = u * c.y + v * c.x;
        }
      }
    }
    void *dst;
    long long at;
    if (is_q) {
      dst = a.q_out, at = (row0 + i) * a.ldqo + (long long)h * a.hd;
    } else if (APPEND) {
      if (slot_i < 0) continue;
      dst = is_v ? a.c.v_pool : a.c.k_pool;
      at = slot_i + (long long)h * a.c.page_size * a.hd;
    } else {
      dst = a.k_out, at = (row0 + i) * a.ldko + (long long)h * a.hd;
    }
    st8<TO>(dst, at + k.dA, x);
    st8<TO>(dst, at + k.dB, x + 8);
  }
}

// Whether CTAs of four rows are the quicker ones: rows in and out of 16 bits, each
// head turned as a whole in halves, head_dim up to 128, CTAs of 128 threads and
// more, and of them six times the 740 that fit the GPU at once. From there on four rows share
// the angles, which one row's threads wait for. Measured in graphs over 400 MB
// and more, heads x head_dim: rows, us for one row | four: 72 x 128: 6,000, 47.8 |
// 45.8; 8,192, 65.3 | 60.6; 32,768, 249 | 220. 72 x 64: 12,000, 48.3 | 44.9. 72 x
// 96: 8,192, 61.4 | 55.4. 40 x 128: 12,000, 52.0 | 50.5; 32,768, 134 | 125. 32 x
// 128: 13,000, 44.9 | 44.2. 32 x 64: 32,768, 53.3 | 49.2. 288 x 128: 2,048, 63.5 |
// 60.2; without norms 72 x 128: 8,192, 55.1 | 48.2. On the other side, 72 x 128
// but for what is said: 2,048 rows, 18.2 | 19.5; 4,096, 33.1 | 32.8; 40 x 128: 8,192,
// 35.9 | 36.0; pairs side by side: 8,192, 77.9 | 91.4; norms alone: 67.1 | 88.0;
// 64 of 128 dims turned: 70.3 | 72.6; to float32: 80.4 | 79.7, 32 heads of 32,768
// rows 137 | 144; 40 x 256: 16,384, 144 | 146; 4 x 128 (CTAs of 32 threads): 131,072, 77.8 | 82.7.
bool four_rows(const RowArgs &a, int threads, int slices) {
  return a.halves && a.dims == a.hd && a.hd <= 128 && threads >= 128 && (long long)(a.rows + 3) / 4 * slices >= 6 * 740;
}

template <int I, int O, bool APPEND>
int launch_types(const RowArgs &a, cudaStream_t st, const char *what) {
  // a task to a thread: slices of the heads beside one another
  const int tasks = (a.nq + a.nk + a.nv) << a.lph_log2, slices = (tasks + kMaxThreads - 1) / kMaxThreads;
  const int threads = ((tasks + slices - 1) / slices + 31) / 32 * 32;
  if constexpr (!APPEND && I != GB_F32 && O != GB_F32) {
    constexpr int R = 4;
    if (four_rows(a, threads, slices)) {
      const int smem = R * threads * 2 * (int)sizeof(Raw<I>);
      GB_CUDA(cudaFuncSetAttribute(head_rows_kernel<I, O, APPEND, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), what);
      head_rows_kernel<I, O, APPEND, R>
          <<<dim3((unsigned)((a.rows + R - 1) / R), (unsigned)slices), (unsigned)threads, smem, st>>>(a);
      GB_CUDA(cudaGetLastError(), what);
      return GB_OK;
    }
  }
  head_rows_kernel<I, O, APPEND, 1><<<dim3((unsigned)a.rows, (unsigned)slices), (unsigned)threads, 0, st>>>(a);
  GB_CUDA(cudaGetLastError(), what);
  return GB_OK;
}

template <bool APPEND>
int launch(const RowArgs &a, int ti, int to, cudaStream_t st, const char *what) {
#define GB_ROWS(I, O) \
  if (ti == I && to == O) return launch_types<I, O, APPEND>(a, st, what);
  GB_ROWS(GB_F32, GB_F32)
  GB_ROWS(GB_F32, GB_F16)
  GB_ROWS(GB_F32, GB_BF16)
  GB_ROWS(GB_F16, GB_F32)
  GB_ROWS(GB_F16, GB_F16)
  GB_ROWS(GB_F16, GB_BF16)
  GB_ROWS(GB_BF16, GB_F32)
  GB_ROWS(GB_BF16, GB_F16)
  GB_ROWS(GB_BF16, GB_BF16)
#undef GB_ROWS
  return gb_fail(GB_ERR_UNSUPPORTED, "%s: types %d and %d", what, ti, to);
}

bool known(int t) { return t == GB_F32 || t == GB_F16 || t == GB_BF16; }

// One operand: a pointer on a 16-byte boundary and rows a multiple of 8 elements apart.
int check_rows(const char *what, const char *name, const void *p, long long ld, int heads, int hd, int rows) {
  if (!p) return gb_fail(GB_ERR_INVALID, "%s: %s is null", what, name);
  if ((uintptr_t)p & 15) return gb_fail(GB_ERR_INVALID, "%s: %s is not on a 16-byte boundary", what, name);
  if (ld % 8 || (rows > 1 && ld < (long long)heads * hd))
    return gb_fail(GB_ERR_INVALID, "%s: %s rows %lld elements apart (a multiple of 8, at least %lld)", what, name, ld,
                   (long long)heads * hd);
  return GB_OK;
}

// What both entry points share: the shapes, the rotation and the norm.
int common(const char *what, RowArgs &a, int nq, int nk, int nv, int hd, int rows, const gb_qk_norm_params *norm,
           const gb_rope_params *rope) {
  if (rows < 0) return gb_fail(GB_ERR_INVALID, "%s: %d rows", what, rows);
  if (rows > (1 << 30)) return gb_fail(GB_ERR_UNSUPPORTED, "%s: %d rows", what, rows);  // rows are counted in 32 bits
  if (nq < 0 || nk < 0 || nq > (1 << 16) || nk > (1 << 16))
    return gb_fail(GB_ERR_INVALID, "%s: %d query heads, %d key heads", what, nq, nk);
  if (hd < 16 || hd > kMaxHD || hd % 16)
    return gb_fail(GB_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 16 up to %d)", what, hd, kMaxHD);
  a.nq = nq, a.nk = nk, a.nv = nv, a.hd = hd, a.rows = rows;
  a.lph_log2 = 0;
  while ((16 << a.lph_log2) < hd) a.lph_log2++;
  if (rope && rope->dims) {
    if (rope->dims < 0 || rope->dims > hd || rope->dims % 16)
      return gb_fail(GB_ERR_UNSUPPORTED, "%s: %d rotated dims of %d (a multiple of 16)", what, rope->dims, hd);
    if (!(rope->base > 0.f) || isinf(rope->base)) return gb_fail(GB_ERR_INVALID, "%s: base %g", what, rope->base);
    a.dims = rope->dims;
    a.halves = rope->halves != 0;
    a.freq = rope->freq;
    a.log2_step = -2.0 * log2((double)rope->base) / rope->dims;
  }
  if (norm) {
    if (!(norm->eps >= 0.f)) return gb_fail(GB_ERR_INVALID, "%s: eps %g", what, norm->eps);
    if (((uintptr_t)norm->wq | (uintptr_t)norm->wk) & 15)
      return gb_fail(GB_ERR_INVALID, "%s: norm weights are not on a 16-byte boundary", what);
    a.wq = norm->wq, a.wk = norm->wk, a.eps = norm->eps;
  }
  return GB_OK;
}

#define GB_TRY(call)              \
  do {                            \
    const int rc_ = (call);       \
    if (rc_ != GB_OK) return rc_; \
  } while (0)

}  // namespace

int gb_qk_norm_rope_launch(int typ, const void *q, long long ldq, int n_heads, const void *k, long long ldk, int n_kv,
                           int rows, int head_dim, const gb_qk_norm_params *norm, const gb_rope_params *rope,
                           const int32_t *pos, int out_typ, void *q_out, long long ldqo, void *k_out, long long ldko,
                           bool loaded, cudaStream_t st) {
  const char *what = "gpu: norm and RoPE";
  RowArgs a = {};
  GB_TRY(common(what, a, n_heads, n_kv, 0, head_dim, rows, norm, rope));
  if (!known(typ) || !known(out_typ)) return gb_fail(GB_ERR_UNSUPPORTED, "%s: types %d and %d", what, typ, out_typ);
  if (rows && a.dims && !pos) return gb_fail(GB_ERR_INVALID, "%s: pos is null", what);
  if (rows && n_heads) {
    GB_TRY(check_rows(what, "q", q, ldq, n_heads, head_dim, rows));
    GB_TRY(check_rows(what, "q_out", q_out, ldqo, n_heads, head_dim, rows));
  }
  if (rows && n_kv) {
    GB_TRY(check_rows(what, "k", k, ldk, n_kv, head_dim, rows));
    GB_TRY(check_rows(what, "k_out", k_out, ldko, n_kv, head_dim, rows));
  }
  if (!loaded) return gb_fail(GB_ERR_INVALID, "gpu: kernels not loaded");
  if (!rows || !(n_heads + n_kv)) return GB_OK;
  a.q = q, a.k = k, a.q_out = q_out, a.k_out = k_out;
  a.ldq = ldq, a.ldk = ldk, a.ldqo = ldqo, a.ldko = ldko;
  a.pos = pos;
  return launch<false>(a, typ, out_typ, st, what);
}

int gb_paged_chunk_check(const char *what, const gb_paged_chunk *c) {
  if (!c) return gb_fail(GB_ERR_INVALID, "%s: no chunk", what);
  if (c->rows < 0 || c->batch < 0 || c->max_pages <= 0 || c->n_pages <= 0 || c->page_size <= 0 || c->n_kv <= 0 ||
      c->n_kv > (1 << 16) || (gb_paged_chunk_any(c) && (!c->q_start || !c->kv_lens || !c->block_table)))
    return gb_fail(GB_ERR_INVALID, "%s: bad arguments", what);
  if ((long long)c->max_pages * c->page_size > 0x7FFFFF00LL)
    return gb_fail(GB_ERR_INVALID, "%s: %d pages of %d positions for a sequence", what, c->max_pages, c->page_size);
  if (!known(c->kv_typ)) return gb_fail(GB_ERR_UNSUPPORTED, "%s: pool type %d", what, c->kv_typ);
  if ((gb_paged_chunk_any(c) && (!c->k_pool || !c->v_pool)) || (((uintptr_t)c->k_pool | (uintptr_t)c->v_pool) & 15))
    return gb_fail(GB_ERR_INVALID, "%s: pools are null or not on a 16-byte boundary", what);
  return GB_OK;
}

int gb_rope_append_paged_launch(const gb_paged_chunk *c, int typ, const void *q, long long ldq, int n_heads,
                                const void *k, long long ldk, const void *v, long long ldv,
                                const gb_qk_norm_params *norm, const gb_rope_params *rope, void *q_out, long long ldqo,
                                bool loaded, cudaStream_t st) {
  const char *what = "gpu: paged append";
  GB_TRY(gb_paged_chunk_check(what, c));
  RowArgs a = {};
  GB_TRY(common(what, a, n_heads, c->n_kv, c->n_kv, c->head_dim, c->rows, norm, rope));
  if (!known(typ)) return gb_fail(GB_ERR_UNSUPPORTED, "%s: type %d", what, typ);
  const bool any = gb_paged_chunk_any(c);
  if (any && n_heads) {
    GB_TRY(check_rows(what, "q", q, ldq, n_heads, c->head_dim, c->rows));
    GB_TRY(check_rows(what, "q_out", q_out, ldqo, n_heads, c->head_dim, c->rows));
  }
  if (any) {
    GB_TRY(check_rows(what, "k", k, ldk, c->n_kv, c->head_dim, c->rows));
    GB_TRY(check_rows(what, "v", v, ldv, c->n_kv, c->head_dim, c->rows));
  }
  if (!loaded) return gb_fail(GB_ERR_INVALID, "gpu: kernels not loaded");
  if (!any) return GB_OK;
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldqo = ldqo;
  a.c = *c;
  return launch<true>(a, typ, c->kv_typ, st, what);
}
