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
constexpr int kMaxThreads = 512;  // threads of a CTA

struct RowArgs {
  const void *q, *k, *v;  // rows of n_heads / n_kv / n_kv heads (v only for the append)
  void *q_out, *k_out;    // k_out only without the append
  long long ldq, ldk, ldv, ldqo, ldko;  // elements between rows
  int nq, nk, nv;         // heads of q, k, v
  int hd, dims, halves;
  int lph_log2;           // lanes per head (16 elements a lane)
  const float *wq, *wk, *freq;
  float eps;
  double log2_base;
  const int32_t *pos;     // without the append
  gb_paged_chunk c;       // with the append
};

template <int T>
GB_DEV void ld8(const void *base, long long i, float *o) {
  if constexpr (T == GB_F32) {
    const float4 x = *(const float4 *)((const float *)base + i), y = *(const float4 *)((const float *)base + i + 4);
    o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w, o[4] = y.x, o[5] = y.y, o[6] = y.z, o[7] = y.w;
  } else {
    const uint4 u = *(const uint4 *)((const uint16_t *)base + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
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

template <int TI>
GB_DEV void task_load(const RowArgs &a, const Task &k, long long row, float *x) {
  if (!k.on) {
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = 0.f;
    return;
  }
  const void *p;
  long long at;
  if (k.head < a.nq) p = a.q, at = row * a.ldq + (long long)k.head * a.hd;
  else if (k.head < a.nq + a.nk) p = a.k, at = row * a.ldk + (long long)(k.head - a.nq) * a.hd;
  else p = a.v, at = row * a.ldv + (long long)(k.head - a.nq - a.nk) * a.hd;
  ld8<TI>(p, at + k.dA, x);
  ld8<TI>(p, at + k.dB, x + 8);
}

// One CTA per row; thread t takes the tasks t, t + blockDim, ... of the row's
// heads. The first task's elements are in flight while the row's sequence is
// looked up and the dims/2 angles are formed once for all heads.
template <int TI, int TO, bool APPEND>
__global__ void __launch_bounds__(kMaxThreads) head_rows_kernel(const __grid_constant__ RowArgs a) {
  __shared__ float2 cs[kMaxHD / 2];
  __shared__ int seq;
  const int row = blockIdx.x, tid = threadIdx.x;
  const int tasks = (a.nq + a.nk + a.nv) << a.lph_log2;
  float x[16];
  Task k = task_of(a, tid);
  task_load<TI>(a, k, row, x);
  long long p;
  long long slot = 0;   // element index of the appended row in head 0 of its page
  bool stored = false;  // the row has a place in the pools
  if constexpr (APPEND) {
    if (tid == 0) seq = a.c.batch;
    __syncthreads();
    for (int b = tid; b < a.c.batch; b += blockDim.x)
      if (a.c.q_start[b] <= row && row < a.c.q_start[b + 1]) atomicMin(&seq, b);
    __syncthreads();
    const int b = seq;
    if (b >= a.c.batch) return;  // a row of no sequence stays as it is
    p = (long long)a.c.kv_lens[b] - a.c.q_start[b + 1] + row;
    if (p >= 0 && p < (long long)a.c.max_pages * a.c.page_size) {
      const int page = a.c.block_table[(long long)b * a.c.max_pages + p / a.c.page_size];
      stored = page >= 0 && page < a.c.n_pages;
      slot = ((long long)page * a.c.n_kv * a.c.page_size + p % a.c.page_size) * a.hd;
    }
  } else {
    p = a.pos ? a.pos[row] : 0;
  }
  for (int j = tid; j < a.dims / 2; j += blockDim.x) {
    double turns = (double)p * exp2(a.log2_base * (-2.0 * j / a.dims)) * 0.15915494309189535;  // 1 / (2 pi)
    if (a.freq) turns /= (double)a.freq[j];
    sincospif((float)(2.0 * (turns - rint(turns))), &cs[j].y, &cs[j].x);
  }
  __syncthreads();
  for (int t = tid;;) {
    const bool is_q = k.head < a.nq, is_v = k.head >= a.nq + a.nk;
    const float *w = is_q ? a.wq : is_v ? nullptr : a.wk;
    // the lanes of a head sit in one warp and agree on w, but a warp's heads may
    // differ: the sum is formed by all lanes, and used where there is a weight
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 16; e++) ss = fmaf(x[e], x[e], ss);
    for (int o = 1; o < (1 << a.lph_log2); o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (k.on) {
      if (w) {
        const float r = rsqrtf(ss / (float)a.hd + a.eps);
        float wv[16];
        ld8<GB_F32>(w, k.dA, wv);
        ld8<GB_F32>(w, k.dB, wv + 8);
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = x[e] * r * wv[e];
      }
      if (k.rot) {
        if (a.halves) {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float2 c = cs[k.dA + e];
            const float u = x[e], v = x[e + 8];
            x[e] = u * c.x - v * c.y;
            x[e + 8] = u * c.y + v * c.x;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float2 c = cs[k.dA / 2 + e];
            const float u = x[2 * e], v = x[2 * e + 1];
            x[2 * e] = u * c.x - v * c.y;
            x[2 * e + 1] = u * c.y + v * c.x;
          }
        }
      }
      void *dst;
      long long at;
      if (is_q) {
        dst = a.q_out, at = (long long)row * a.ldqo + (long long)k.head * a.hd;
      } else if (APPEND) {
        dst = is_v ? a.c.v_pool : a.c.k_pool;
        const int h = k.head - a.nq - (is_v ? a.nk : 0);
        at = slot + (long long)h * a.c.page_size * a.hd;
      } else {
        dst = a.k_out, at = (long long)row * a.ldko + (long long)(k.head - a.nq) * a.hd;
      }
      if (is_q || !APPEND || stored) {
        st8<TO>(dst, at + k.dA, x);
        st8<TO>(dst, at + k.dB, x + 8);
      }
    }
    t += blockDim.x;
    if ((t & ~31) >= tasks) break;  // a whole warp leaves together
    k = task_of(a, t);
    task_load<TI>(a, k, row, x);
  }
}

template <bool APPEND>
int launch(const RowArgs &a, int rows, int ti, int to, cudaStream_t st, const char *what) {
  const int tasks = (a.nq + a.nk + a.nv) << a.lph_log2;
  const int turns = (tasks + kMaxThreads - 1) / kMaxThreads;
  const int threads = ((tasks + turns - 1) / turns + 31) / 32 * 32;
#define GB_ROWS(I, O)                                                              \
  if (ti == I && to == O) {                                                        \
    head_rows_kernel<I, O, APPEND><<<(unsigned)rows, (unsigned)threads, 0, st>>>(a); \
    GB_CUDA(cudaGetLastError(), what);                                             \
    return GB_OK;                                                                  \
  }
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
  if (nq < 0 || nk < 0 || nq > (1 << 16) || nk > (1 << 16))
    return gb_fail(GB_ERR_INVALID, "%s: %d query heads, %d key heads", what, nq, nk);
  if (hd < 16 || hd > kMaxHD || hd % 16)
    return gb_fail(GB_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 16 up to %d)", what, hd, kMaxHD);
  a.nq = nq, a.nk = nk, a.nv = nv, a.hd = hd;
  a.lph_log2 = 0;
  while ((16 << a.lph_log2) < hd) a.lph_log2++;
  if (rope && rope->dims) {
    if (rope->dims < 0 || rope->dims > hd || rope->dims % 16)
      return gb_fail(GB_ERR_UNSUPPORTED, "%s: %d rotated dims of %d (a multiple of 16)", what, rope->dims, hd);
    if (!(rope->base > 0.f) || isinf(rope->base)) return gb_fail(GB_ERR_INVALID, "%s: base %g", what, rope->base);
    a.dims = rope->dims;
    a.halves = rope->halves != 0;
    a.freq = rope->freq;
    a.log2_base = log2((double)rope->base);
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
  if (a.dims && !pos) return gb_fail(GB_ERR_INVALID, "%s: pos is null", what);
  if (n_heads) {
    GB_TRY(check_rows(what, "q", q, ldq, n_heads, head_dim, rows));
    GB_TRY(check_rows(what, "q_out", q_out, ldqo, n_heads, head_dim, rows));
  }
  if (n_kv) {
    GB_TRY(check_rows(what, "k", k, ldk, n_kv, head_dim, rows));
    GB_TRY(check_rows(what, "k_out", k_out, ldko, n_kv, head_dim, rows));
  }
  if (!loaded) return gb_fail(GB_ERR_INVALID, "gpu: kernels not loaded");
  if (!rows || !(n_heads + n_kv)) return GB_OK;
  a.q = q, a.k = k, a.q_out = q_out, a.k_out = k_out;
  a.ldq = ldq, a.ldk = ldk, a.ldqo = ldqo, a.ldko = ldko;
  a.pos = pos;
  return launch<false>(a, rows, typ, out_typ, st, what);
}

int gb_paged_chunk_check(const char *what, const gb_paged_chunk *c) {
  if (!c) return gb_fail(GB_ERR_INVALID, "%s: no chunk", what);
  if (c->rows < 0 || c->batch < 0 || c->max_pages <= 0 || c->n_pages <= 0 || c->page_size <= 0 || c->n_kv <= 0 ||
      c->n_kv > (1 << 16) || !c->q_start || !c->kv_lens || !c->block_table)
    return gb_fail(GB_ERR_INVALID, "%s: bad arguments", what);
  if ((long long)c->max_pages * c->page_size > 0x7FFFFF00LL)
    return gb_fail(GB_ERR_INVALID, "%s: %d pages of %d positions for a sequence", what, c->max_pages, c->page_size);
  if (!known(c->kv_typ)) return gb_fail(GB_ERR_UNSUPPORTED, "%s: pool type %d", what, c->kv_typ);
  if (!c->k_pool || !c->v_pool || (((uintptr_t)c->k_pool | (uintptr_t)c->v_pool) & 15))
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
  if (n_heads) {
    GB_TRY(check_rows(what, "q", q, ldq, n_heads, c->head_dim, c->rows));
    GB_TRY(check_rows(what, "q_out", q_out, ldqo, n_heads, c->head_dim, c->rows));
  }
  GB_TRY(check_rows(what, "k", k, ldk, c->n_kv, c->head_dim, c->rows));
  GB_TRY(check_rows(what, "v", v, ldv, c->n_kv, c->head_dim, c->rows));
  if (!loaded) return gb_fail(GB_ERR_INVALID, "gpu: kernels not loaded");
  if (!c->rows || !c->batch) return GB_OK;
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldqo = ldqo;
  a.c = *c;
  return launch<true>(a, c->rows, typ, c->kv_typ, st, what);
}
