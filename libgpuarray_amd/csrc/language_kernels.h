/* Kernels of the operators in gpuarray/language.h, for 64-lane wavefronts.
 *
 * The text is compiled at run time, one operator and one set of types at a
 * time, behind these #defines:
 *   LM_KIND   which operator, LM_K_* below
 *   LM_X      element type of the operand (table, logits, dout)
 *   LM_O      element type of the result (rows, gradient of the table)
 *   LM_ID     type of the ids
 * and, per operator, the variant's own.  Arguments travel in one struct by
 * value, with plain device addresses; strides are in bytes.
 *
 * Ids: an id that is `ignore` stands for no token; a negative one counts from
 * the end; one out of range sets the error word and touches nothing. */
#include "cluda.h"

#define LM_K_EMBED 0
#define LM_K_EMBED_GRAD 1
#define LM_K_LOGPROBS 2
#define LM_K_LOGPROBS_GRAD 3
#define LM_K_NORM 4
#define LM_K_CLIP 5

#define LM_FN static __device__ __forceinline__

LM_FN float lm_get(ga_float x) { return x; }
LM_FN float lm_get(ga_half x) { return ga_half2float(x); }
LM_FN float lm_get(ga_bfloat16 x) { return x; }
LM_FN double lm_get(ga_double x) { return x; }
LM_FN void lm_put(ga_float *p, float v) { *p = v; }
LM_FN void lm_put(ga_half *p, float v) { *p = ga_float2half(v); }
LM_FN void lm_put(ga_bfloat16 *p, float v) { *p = ga_bfloat16(v); }
LM_FN void lm_put(ga_double *p, double v) { *p = v; }

template <class T> LM_FN T *lm_at(T *base, ga_long bytes) {
  return (T *)((GLOBAL_MEM char *)base + bytes);
}

/* An id in [0, v); -1: no token; -2: out of range. */
LM_FN ga_long lm_id(ga_long id, ga_long ignore, ga_long none, ga_long v) {
  if (ignore != none && id == ignore) return -1;
  if (id < 0) id += v;
  return id >= 0 && id < v ? id : -2;
}
/* the value of ignore that no id is compared with */
#define LM_NONE ((ga_long)1 << 63)

LM_FN float lm_wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute((int)(((LID_0 & 63) ^ d) << 2), __builtin_bit_cast(int, v)));
  return v;
}
LM_FN float lm_wave_max(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = __builtin_fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute((int)(((LID_0 & 63) ^ d) << 2), __builtin_bit_cast(int, v))));
  return v;
}

#if LM_KIND == LM_K_EMBED
struct lm_embed {
  GLOBAL_MEM LM_O *out;
  GLOBAL_MEM const LM_X *table;
  GLOBAL_MEM const LM_ID *ids;
  GLOBAL_MEM ga_int *err;
  ga_long out_row, table_row, id_step;
  ga_long n, v, d, ignore;
  float scale;
};
KERNEL void __launch_bounds__(256) lm_embed_rows(const lm_embed p) {
  const ga_long row = GID_0;
  const ga_long id = lm_id((ga_long)*lm_at(p.ids, row * p.id_step), p.ignore, LM_NONE, p.v);
  if (id == -2) {
    if (LID_0 == 0) *p.err = -1;
    return;
  }
  GLOBAL_MEM LM_O *o = lm_at(p.out, row * p.out_row);
  GLOBAL_MEM const LM_X *x = lm_at(p.table, id * p.table_row);
  for (ga_long c = LID_0; c < p.d; c += 256) lm_put(o + c, id < 0 ? 0.0f : p.scale * lm_get(x[c]));
}
#endif

#if LM_KIND == LM_K_EMBED_GRAD
struct lm_embed_grad {
  GLOBAL_MEM LM_O *grad;
  GLOBAL_MEM const LM_X *dout;
  GLOBAL_MEM const LM_ID *ids;
  GLOBAL_MEM ga_int *err;
  ga_long grad_row, dout_row, id_step;
  ga_long n, v, d, ignore;
  float scale;
  ga_int accumulate;
};
/* One wavefront per row of the table: it looks through all ids for its own and
 * adds the rows of dout that have it, in order. */
KERNEL void __launch_bounds__(256) lm_embed_grad_rows(const lm_embed_grad p) {
  const ga_long r = (ga_long)GID_0 * 4 + (LID_0 >> 6);
  const ga_uint lane = LID_0 & 63;
  if (r >= p.v && r != 0) return;   /* (row 0 also looks for ids out of range) */
  for (ga_long c0 = 0; c0 < p.d || c0 == 0; c0 += 512) {
    float sum[8];
    bool any = false;
#pragma unroll
    for (int u = 0; u < 8; u++) sum[u] = 0.0f;
    for (ga_long base = 0; base < p.n; base += 64) {
      const ga_long i = base + lane;
      const ga_long id = i < p.n ? lm_id((ga_long)*lm_at(p.ids, i * p.id_step), p.ignore, LM_NONE, p.v) : -1;
      if (id == -2 && r == 0) *p.err = -1;
      ga_ulong hits = __builtin_amdgcn_ballot_w64(id == r);
      any = any || hits != 0;
      while (hits != 0) {
        const ga_long at = base + __builtin_ctzll(hits);
        hits &= hits - 1;
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const ga_long c = c0 + u * 64 + lane;
          if (c < p.d) sum[u] += lm_get(lm_at(p.dout, at * p.dout_row)[c]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const ga_long c = c0 + u * 64 + lane;
      GLOBAL_MEM LM_O *g = lm_at(p.grad, r * p.grad_row) + c;
      if (c < p.d && r < p.v) {
        if (!p.accumulate) lm_put(g, p.scale * sum[u]);
        else if (any) lm_put(g, lm_get(*g) + p.scale * sum[u]);
      }
    }
  }
}
#endif

#if LM_KIND == LM_K_LOGPROBS
struct lm_logprobs {
  GLOBAL_MEM const LM_X *logits;
  GLOBAL_MEM const LM_ID *ids;   /* NULL: no logp */
  GLOBAL_MEM float *logp, *entropy, *stats, *top_logp;   /* NULL: not wanted */
  GLOBAL_MEM void *top_ids;
  GLOBAL_MEM ga_int *err;
  ga_long row, id_step, logp_step, entropy_step, stats_row, stats_col;
  ga_long topl_row, topl_col, topi_row, topi_col;
  ga_long t, v, ignore;
  float scale;
  ga_int top, top_long;
};

/* what is written for row r, from its statistics; one lane */
LM_FN void lm_logprobs_finish(const lm_logprobs &p, ga_long r, float m, float ls, float entropy) {
  if (p.ids != nullptr) {
    const ga_long id = lm_id((ga_long)*lm_at(p.ids, r * p.id_step), p.ignore, LM_NONE, p.v);
    float lp = 0.0f;
    if (id == -2) {
      *p.err = -1;
      lp = NAN;
    } else if (id >= 0) {
      lp = ls == -INFINITY ? -INFINITY : (lm_get(lm_at(p.logits, r * p.row)[id]) - m) * p.scale - ls;
      if (ls != ls) lp = NAN;
    }
    *lm_at(p.logp, r * p.logp_step) = lp;
  }
  if (p.entropy != nullptr) *lm_at(p.entropy, r * p.entropy_step) = ls == -INFINITY ? 0.0f : entropy;
  if (p.stats != nullptr) {
    *lm_at(p.stats, r * p.stats_row) = m;
    *lm_at(p.stats, r * p.stats_row + p.stats_col) = ls;
  }
}
LM_FN void lm_put_top(const lm_logprobs &p, ga_long r, ga_int k, float lp, ga_long id) {
  *lm_at(p.top_logp, r * p.topl_row + k * p.topl_col) = lp;
  const ga_long at = r * p.topi_row + k * p.topi_col;
  if (p.top_long) *lm_at((GLOBAL_MEM ga_long *)p.top_ids, at) = id;
  else *lm_at((GLOBAL_MEM ga_int *)p.top_ids, at) = (ga_int)id;
}

/* One wavefront per row, in passes: the maximum; the sums; then one pass for
 * each alternative, the largest value after the one before it. */
KERNEL void __launch_bounds__(64) lm_logprobs_rows(const lm_logprobs p) {
  const ga_long r = GID_0;
  const ga_uint lane = LID_0;
  GLOBAL_MEM const LM_X *x = lm_at(p.logits, r * p.row);
  float m = -INFINITY;
  for (ga_long c = lane; c < p.v; c += 64) m = __builtin_fmaxf(m, lm_get(x[c]));
  m = lm_wave_max(m);
  const float m0 = m == -INFINITY ? 0.0f : m;
  float s = 0.0f, w = 0.0f;
  for (ga_long c = lane; c < p.v; c += 64) {
    const float z = (lm_get(x[c]) - m0) * p.scale, e = __builtin_expf(z);
    s += e;
    w += e * __builtin_fmaxf(z, -1000.0f);
  }
  s = lm_wave_sum(s);
  w = lm_wave_sum(w);
  const float ls = __builtin_logf(s);
  if (lane == 0) lm_logprobs_finish(p, r, m, ls, ls - w / s);
  float lv = INFINITY;
  ga_int li = -1;
  for (ga_int k = 0; k < p.top; k++) {
    if (ls != ls) {
      if (lane == 0) lm_put_top(p, r, k, NAN, k);
      continue;
    }
    float bv = -INFINITY;
    ga_int bi = 0x7fffffff;
    for (ga_int c = lane; c < p.v; c += 64) {
      const float y = lm_get(x[c]);
      if ((y < lv || (y == lv && c > li)) && (y > bv || bi == 0x7fffffff)) {
        bv = y;
        bi = c;
      }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const int from = (int)((lane ^ d) << 2);
      const float ov = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(from, __builtin_bit_cast(int, bv)));
      const ga_int oi = __builtin_amdgcn_ds_bpermute(from, bi);
      if (ov > bv || (ov == bv && oi < bi)) {
        bv = ov;
        bi = oi;
      }
    }
    if (lane == 0) lm_put_top(p, r, k, ls == -INFINITY ? -INFINITY : (bv - m) * p.scale - ls, bi);
    lv = bv;
    li = bi;
  }
}
#endif

#if LM_KIND == LM_K_LOGPROBS_GRAD
struct lm_logprobs_grad {
  GLOBAL_MEM LM_X *out;
  GLOBAL_MEM const LM_X *logits;
  GLOBAL_MEM const LM_ID *ids;   /* NULL: no gradient of logp */
  GLOBAL_MEM const float *stats, *dlogp, *entropy, *dentropy;
  GLOBAL_MEM ga_int *err;
  ga_long out_row, row, id_step, stats_row, stats_col, dlogp_step, entropy_step, dentropy_step;
  ga_long t, v, ignore;
  float scale;
};
KERNEL void __launch_bounds__(256) lm_logprobs_grad_rows(const lm_logprobs_grad p) {
  const ga_long r = GID_0;
  GLOBAL_MEM const LM_X *x = lm_at(p.logits, r * p.row);
  GLOBAL_MEM LM_X *o = lm_at(p.out, r * p.out_row);
  const float m = *lm_at(p.stats, r * p.stats_row), ls = *lm_at(p.stats, r * p.stats_row + p.stats_col);
  float g = 0.0f, gh = 0.0f, h = 0.0f;
  ga_long id = -1;
  if (p.ids != nullptr) {
    id = lm_id((ga_long)*lm_at(p.ids, r * p.id_step), p.ignore, LM_NONE, p.v);
    if (id == -2 && LID_0 == 0) *p.err = -1;
    if (id >= 0) g = *lm_at(p.dlogp, r * p.dlogp_step);
  }
  if (p.entropy != nullptr) {
    gh = *lm_at(p.dentropy, r * p.dentropy_step);
    h = *lm_at(p.entropy, r * p.entropy_step);
  }
  for (ga_long c = LID_0; c < p.v; c += 256) {
    float d = 0.0f;
    if (ls != -INFINITY) {
      const float lp = (lm_get(x[c]) - m) * p.scale - ls, q = __builtin_expf(lp);
      d = p.scale * ((c == id ? g : 0.0f) - q * (g + gh * (__builtin_fmaxf(lp, -1000.0f) + h)));
    }
    lm_put(o + c, d);
  }
}
#endif

#if LM_KIND == LM_K_NORM || LM_KIND == LM_K_CLIP
/* The arrays of a launch: up to LM_TENSORS of them, cut in pieces of LM_PIECE
 * elements that are numbered through; first[i] is the number of array i's
 * first piece.  The count of arrays is small next to the work, so a piece
 * finds its array by bisection of the table in its arguments. */
#define LM_PIECE 8192
struct lm_tensors {
  GLOBAL_MEM double *partials;   /* sums of squares, one per piece */
  GLOBAL_MEM double *result;     /* norm, factor */
  GLOBAL_MEM void *norm;
  double max_norm;
  ga_long partial0, npartials;
  ga_int n, norm_double, clip, pad;
  GLOBAL_MEM const void *in[LM_TENSORS];
  GLOBAL_MEM void *out[LM_TENSORS];
  ga_long count[LM_TENSORS];
  ga_uint first[LM_TENSORS + 1];
  unsigned char type[LM_TENSORS];   /* 0 float, 1 half, 2 bfloat16, 3 double */
};
LM_FN ga_int lm_find(const lm_tensors &p, ga_uint piece) {
  ga_int lo = 0, hi = p.n;
  while (hi - lo > 1) {
    const ga_int mid = (lo + hi) >> 1;
    if (p.first[mid] <= piece) lo = mid;
    else hi = mid;
  }
  return lo;
}
#define LM_BY_TYPE(type, F)                     \
  switch (type) {                               \
    case 0: F(ga_float, float) break;           \
    case 1: F(ga_half, float) break;            \
    case 2: F(ga_bfloat16, float) break;        \
    default: F(ga_double, double) break;        \
  }
/* the sum over a group of 256 lanes, in lane 0 */
LM_FN double lm_group_sum(double v) {
  LOCAL_MEM double part[256];
  part[LID_0] = v;
  local_barrier();
#pragma unroll
  for (int d = 128; d > 0; d >>= 1) {
    if (LID_0 < d) part[LID_0] += part[LID_0 + d];
    local_barrier();
  }
  return part[0];
}
#endif

#if LM_KIND == LM_K_NORM
KERNEL void __launch_bounds__(256) lm_norm_pieces(const lm_tensors p) {
  const ga_int i = lm_find(p, GID_0);
  const ga_long from = (ga_long)(GID_0 - p.first[i]) * LM_PIECE;
  const ga_long left = p.count[i] - from;
  const ga_int n = left < LM_PIECE ? (ga_int)left : LM_PIECE;
  double s = 0.0;
#define LM_SQUARES(T, A)                                        \
  for (ga_int k = LID_0; k < n; k += 256) {                     \
    const double x = lm_get(((GLOBAL_MEM const T *)p.in[i])[from + k]); \
    s += x * x;                                                 \
  }
  LM_BY_TYPE(p.type[i], LM_SQUARES)
  s = lm_group_sum(s);
  if (LID_0 == 0) p.partials[p.partial0 + GID_0] = s;
}
KERNEL void __launch_bounds__(256) lm_norm_final(const lm_tensors p) {
  double s = 0.0;
  for (ga_long k = LID_0; k < p.npartials; k += 256) s += p.partials[k];
  s = lm_group_sum(s);
  if (LID_0 == 0) {
    const double norm = __builtin_sqrt(s);
    p.result[0] = norm > p.max_norm && norm < (double)INFINITY ? p.max_norm / norm : 1.0;
    if (p.norm != nullptr) {
      if (p.norm_double) *(GLOBAL_MEM double *)p.norm = norm;
      else *(GLOBAL_MEM float *)p.norm = (float)norm;
    }
  }
}
#endif

#if LM_KIND == LM_K_CLIP
KERNEL void __launch_bounds__(256) lm_clip_pieces(const lm_tensors p) {
  const double by = p.result[0];
  const ga_int i = lm_find(p, GID_0);
  if (by == 1.0 && p.in[i] == p.out[i]) return;
  const ga_long from = (ga_long)(GID_0 - p.first[i]) * LM_PIECE;
  const ga_long left = p.count[i] - from;
  const ga_int n = left < LM_PIECE ? (ga_int)left : LM_PIECE;
#define LM_SCALE(T, A)                                          \
  for (ga_int k = LID_0; k < n; k += 256)                       \
    lm_put((GLOBAL_MEM T *)p.out[i] + from + k, (A)by * lm_get(((GLOBAL_MEM const T *)p.in[i])[from + k]));
  LM_BY_TYPE(p.type[i], LM_SCALE)
}
#endif
