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
#define LM_K_SORT 6

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
template <class T> LM_FN ga_long lm_id(T raw, ga_long ignore, ga_long none, ga_long v) {
  ga_long id = (ga_long)raw;
  if ((T)-1 > (T)0 && id < 0) return -2;   /* an unsigned id of 2^63 or more does not count from the end */
  if (ignore != none && id == ignore) return -1;
  if (id < 0) id += v;
  return id >= 0 && id < v ? id : -2;
}
/* the value of ignore that no id is compared with */
#define LM_NONE ((ga_long)1 << 63)

/* The value of lane ^ MASK: through the data-parallel moves where one of them
 * is that exchange, else through the LDS crossbar. */
template <int MASK> LM_FN ga_uint lm_xor(ga_uint v) {
  if constexpr (MASK == 1) return (ga_uint)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);
  else if constexpr (MASK == 2) return (ga_uint)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);
  else if constexpr (MASK == 3) return (ga_uint)__builtin_amdgcn_update_dpp(0, (int)v, 0x1B, 0xF, 0xF, true);
  else if constexpr (MASK == 7) return (ga_uint)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true);
  else if constexpr (MASK == 8) return (ga_uint)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true);
  else if constexpr (MASK == 15) return (ga_uint)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true);
  else if constexpr (MASK < 32) return (ga_uint)__builtin_amdgcn_ds_swizzle((int)v, (MASK << 10) | 0x1F);
  else return (ga_uint)__builtin_amdgcn_ds_bpermute((int)(((LID_0 & 63) ^ MASK) << 2), (int)v);
}
template <int MASK> LM_FN float lm_xor(float v) {
  return __builtin_bit_cast(float, lm_xor<MASK>(__builtin_bit_cast(ga_uint, v)));
}
template <int MASK> LM_FN ga_ulong lm_xor(ga_ulong v) {
  return (ga_ulong)lm_xor<MASK>((ga_uint)(v >> 32)) << 32 | lm_xor<MASK>((ga_uint)v);
}

/* ---- the group that finishes last finishes the call ---------------------------------
 * Few groups leave partial results with device-scope stores, wait until those
 * are acknowledged (past the L2 of their die) and count themselves in; the one
 * that completes the count fetches all of them, in fixed order, with device-scope
 * loads, and zeroes the counter.  Nobody waits for anybody. */
template <class T> LM_FN void lm_publish(GLOBAL_MEM T *p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T> LM_FN T lm_fetch(GLOBAL_MEM const T *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
/* by the lane, or the wavefront, that published; true for the last of `total` */
LM_FN bool lm_count_in(GLOBAL_MEM ga_uint *counter, ga_uint total) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const bool last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == total;
  if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("" ::: "memory");
  return last;
}

/* ---- 16-byte chunks of a row -------------------------------------------------- */
typedef ga_uint lm_u4 __attribute__((ext_vector_type(4)));
#define LM_E (16 / (int)sizeof(LM_X))   /* elements of a chunk */

LM_FN void lm_unpack(const lm_u4 &q, float *y, ga_float) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const ga_uint word = q[e];   /* (a bit cast of the vector's element itself gives the first one) */
    y[e] = __builtin_bit_cast(float, word);
  }
}
LM_FN void lm_unpack(const lm_u4 &q, float *y, ga_half) {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  const h8 h = __builtin_bit_cast(h8, q);
#pragma unroll
  for (int e = 0; e < 8; e++) y[e] = (float)h[e];
}
LM_FN void lm_unpack(const lm_u4 &q, float *y, ga_bfloat16) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    y[2 * e] = __builtin_bit_cast(float, q[e] << 16);
    y[2 * e + 1] = __builtin_bit_cast(float, q[e] & 0xffff0000u);
  }
}
/* N adjacent elements, 8 or 16 or 32 bytes, from an address that is aligned to
 * the element only; and the same for results. */
typedef ga_uint lm_u2a __attribute__((ext_vector_type(2), aligned(2)));
typedef ga_uint lm_u4a __attribute__((ext_vector_type(4), aligned(2)));
template <int N, class T> LM_FN void lm_load(GLOBAL_MEM const T *p, float (&y)[N]) {
  constexpr int per = 16 / (int)sizeof(T);
  if constexpr (N * sizeof(T) == 8) {
    const lm_u2a q = *(GLOBAL_MEM const lm_u2a *)p;
    const lm_u4 wide = {q[0], q[1], 0, 0};
    float z[8];
    lm_unpack(wide, z, T());
#pragma unroll
    for (int e = 0; e < N; e++) y[e] = z[e];
  } else {
#pragma unroll
    for (int i = 0; i < N / per; i++) {
      const lm_u4 q = *(GLOBAL_MEM const lm_u4a *)(p + i * per);
      lm_unpack(q, y + i * per, T());
    }
  }
}
LM_FN ga_uint lm_pair(float a, float b, ga_half) {
  return (ga_uint)ga_float2half(a).data | (ga_uint)ga_float2half(b).data << 16;
}
LM_FN ga_uint lm_pair(float a, float b, ga_bfloat16) {   /* one conversion instruction for both */
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  const b2 r = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(ga_uint, r);
}
LM_FN void lm_pack(const float *y, ga_uint *w, int n, ga_float) {
#pragma unroll
  for (int i = 0; i < n; i++) w[i] = __builtin_bit_cast(ga_uint, y[i]);
}
template <class T> LM_FN void lm_pack(const float *y, ga_uint *w, int n, T) {
#pragma unroll
  for (int i = 0; i < n; i++) w[i] = lm_pair(y[2 * i], y[2 * i + 1], T());
}
template <int N, class T> LM_FN void lm_store(GLOBAL_MEM T *p, const float (&y)[N]) {
  constexpr int words = N * (int)sizeof(T) / 4;
  ga_uint w[words];
  lm_pack(y, w, words, T());
  if constexpr (words == 2) {
    const lm_u2a q = {w[0], w[1]};
    *(GLOBAL_MEM lm_u2a *)p = q;
  } else {
#pragma unroll
    for (int i = 0; i < words; i += 4) {
      const lm_u4a q = {w[i], w[i + 1], w[i + 2], w[i + 3]};
      /* two halves of 32 bytes are put together by the L2, which a streamed store passes by */
      if constexpr (words == 4) __builtin_nontemporal_store(q, (GLOBAL_MEM lm_u4a *)(p + i * 4 / (int)sizeof(T)));
      else *(GLOBAL_MEM lm_u4a *)(p + i * 4 / (int)sizeof(T)) = q;
    }
  }
}

/* a word of -inf elements */
LM_FN ga_uint lm_minus_inf(ga_float) { return 0xff800000u; }
LM_FN ga_uint lm_minus_inf(ga_half) { return 0xfc00fc00u; }
LM_FN ga_uint lm_minus_inf(ga_bfloat16) { return 0xff80ff80u; }

/* Zeroes `bytes` bytes from b on, whose elements have 2 or 4, by `lanes` lanes (32 or more). */
LM_FN void lm_zero(GLOBAL_MEM char *b, ga_long bytes, ga_uint lane, ga_uint lanes) {
  ga_long head = (ga_long)(-(ga_size)b & 15);
  if (head > bytes) head = bytes;
  const ga_long chunks = (bytes - head) / 16, tail = head + chunks * 16;
  GLOBAL_MEM lm_u4 *q = (GLOBAL_MEM lm_u4 *)(b + head);
  const lm_u4 zero = {0, 0, 0, 0};
  for (ga_long c = lane; c < chunks; c += lanes) __builtin_nontemporal_store(zero, q + c);
  const ga_long at = lane * 2 < head ? lane * 2 : tail + (lane * 2 - head);
  if (at < bytes) *(GLOBAL_MEM ga_ushort *)(b + at) = 0;
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
  ga_uint lanes_log2, segments;
};
#define LM_C (16 / (int)sizeof(LM_O))   /* elements of a lane: 16 bytes of the result */
#define LM_ROWS 4

/* 2^lanes_log2 lanes share a row's 256 * LM_C columns or fewer; a lane moves the
 * same columns of LM_ROWS rows, so that the loads of the ids, of the rows and the
 * stores each go out together.  Bound by memory: 16384 rows of 1024 bfloat16 10.8 us
 * (33 MB out, 19 MB of distinct rows in, 33 asked for), 24211 rows of 6494 bfloat16 as floats 156 us
 * (6.0 TB/s; with 32 bytes of the result a lane 250). */
KERNEL void __launch_bounds__(256) lm_embed_rows(const lm_embed p) {
  const ga_uint lane = LID_0 & ((1u << p.lanes_log2) - 1u), side = 256u >> p.lanes_log2;
  const ga_long row0 = (ga_long)(GID_0 / p.segments) * side * LM_ROWS + (LID_0 >> p.lanes_log2);
  const ga_long col = ((ga_long)(GID_0 % p.segments) * 256 + lane) * LM_C;
  ga_long id[LM_ROWS];
#pragma unroll
  for (int u = 0; u < LM_ROWS; u++) {
    const ga_long row = row0 + u * side;
    id[u] = row < p.n ? lm_id(*lm_at(p.ids, row * p.id_step), p.ignore, LM_NONE, p.v) : -3;
    if (id[u] == -2) *p.err = -1;
  }
  if (col >= p.d) return;
  /* Loads are unconditional, so that all of them are in flight at once: rows
   * of no token fetch row 0, and the lane at a row's end fetches the row's
   * last LM_C columns, of which it writes its own. */
  const ga_long from = p.d >= LM_C && p.d - col < LM_C ? p.d - LM_C : col;
  const ga_int skip = (ga_int)(col - from);
  float y[LM_ROWS][LM_C];
  if (p.d >= LM_C && p.v != 0) {
#pragma unroll
    for (int u = 0; u < LM_ROWS; u++) lm_load(lm_at(p.table, (id[u] > 0 ? id[u] : 0) * p.table_row) + from, y[u]);
  } else {
#pragma unroll
    for (int u = 0; u < LM_ROWS; u++)
#pragma unroll
      for (int e = 0; e < LM_C; e++) {
        const bool in = e < p.d && p.v != 0;
        y[u][e] = in ? (float)lm_get(lm_at(p.table, (id[u] > 0 ? id[u] : 0) * p.table_row)[e]) : 0.0f;
      }
  }
#pragma unroll
  for (int u = 0; u < LM_ROWS; u++) {
    if (id[u] < -1) continue;
    GLOBAL_MEM LM_O *o = lm_at(p.out, (row0 + u * side) * p.out_row) + from;
#pragma unroll
    for (int e = 0; e < LM_C; e++) y[u][e] = id[u] >= 0 ? y[u][e] * p.scale : 0.0f;
    if (skip == 0 && p.d >= LM_C) {
      lm_store(o, y[u]);
    } else {
#pragma unroll
      for (int e = 0; e < LM_C; e++)
        if (e >= skip && from + e < p.d) lm_put(o + e, y[u][e]);
    }
  }
}
#endif

#if LM_KIND == LM_K_SORT
/* ---- tokens in the order of their ids ---------------------------------------------
 * The gradient of the table adds the rows of equal ids, so the tokens are
 * sorted by id first: least significant digit first, every pass stable, so that
 * the tokens of one id stay in their order and sums are the same on every call.
 * No token and out of range become the key v, past all rows.  LM_R items per
 * lane, 1024 lanes per group; an item's place among the equal digits of its
 * wavefront is counted with ballots, one per bit.
 *
 * All that is short next to clearing the gradient's rows, which needs none of
 * it: every launch of the sort has more groups than it needs for that, and those
 * clear a share of the rows meanwhile (8192 ids, 206 MB: 35 us, 5.9 TB/s; the sort
 * alone 17, a fill of as much 30). */
struct lm_sorting {
  GLOBAL_MEM const LM_ID *ids;      /* of the first pass */
  GLOBAL_MEM const ga_uint *key_in, *order_in;
  GLOBAL_MEM ga_uint *key, *order;  /* results of the pass */
  GLOBAL_MEM ga_uint *counts;       /* [digit][group], then [digit] totals; [group][digit] if `direct` */
  GLOBAL_MEM ga_int *err;
  ga_long id_step, ignore, v;
  ga_uint n, groups, shift, bits, passes;
  ga_uint direct;                   /* no lm_sort_scan: every group adds the counts itself */
  GLOBAL_MEM char *fill;            /* rows to clear: */
  ga_long fill_rows, fill_row, fill_bytes, fill_unit0, fill_unit1;
};
#define LM_SEGMENT 16384   /* bytes that a wavefront clears at a time */

/* Units [fill_unit0, fill_unit1) of rows x segments, over the wavefronts of the groups past `first`. */
LM_FN void lm_clear(const lm_sorting &p, ga_uint first) {
  const ga_long segments = (p.fill_bytes + LM_SEGMENT - 1) / LM_SEGMENT;
  const ga_uint lane = LID_0 & 63;
  const ga_long waves = (ga_long)(GDIM_0 - first) * 16;
  for (ga_long u = p.fill_unit0 + (ga_long)(GID_0 - first) * 16 + (LID_0 >> 6); u < p.fill_unit1; u += waves) {
    const ga_long row = u / segments, seg = u % segments;
    const ga_long bytes = p.fill_bytes - seg * LM_SEGMENT;
    lm_zero(p.fill + row * p.fill_row + seg * LM_SEGMENT, bytes < LM_SEGMENT ? bytes : LM_SEGMENT, lane, 64);
  }
}

LM_FN ga_uint lm_first_key(const lm_sorting &p, ga_uint i) {
  const ga_long id = lm_id(*lm_at(p.ids, (ga_long)i * p.id_step), p.ignore, LM_NONE, p.v);
  if (id == -2) *p.err = -1;
  return id < 0 ? (ga_uint)p.v : (ga_uint)id;
}

/* exclusive prefix sum over 1024 lanes */
LM_FN ga_uint lm_scan(ga_uint x) {
  LOCAL_MEM ga_uint sums[16];
  const ga_uint lane = LID_0 & 63, wave = LID_0 >> 6;
  ga_uint s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const ga_uint y = (ga_uint)__builtin_amdgcn_ds_bpermute((int)((lane - d) << 2), (int)s);
    if (lane >= d) s += y;
  }
  if (lane == 63) sums[wave] = s;
  local_barrier();
  ga_uint before = 0;
  for (ga_uint i = 0; i < wave; i++) before += sums[i];
  local_barrier();
  return before + s - x;
}

#define LM_BINS 1024   /* digits of up to 10 bits */
/* rank[r]: how many equal digits this wavefront has before item r of this lane;
 * counts[wave]: how many it has of each digit in all.  Item r of lane l is item r * 64 + l of the
 * wavefront. */
LM_FN void lm_rank(const ga_uint (&k)[LM_R], ga_uint (&rank)[LM_R], volatile ga_ushort (*counts)[LM_BINS],
                   ga_uint shift, ga_uint bits) {
  const ga_uint lane = LID_0 & 63, wave = LID_0 >> 6, mask = (1u << bits) - 1;
  for (ga_uint b = LID_0; b < 16 * LM_BINS / 2; b += 1024) ((volatile ga_uint *)counts)[b] = 0;
  local_barrier();
#pragma unroll
  for (int r = 0; r < LM_R; r++) {
    const ga_uint d = (k[r] >> shift) & mask;
    ga_ulong peers = ~(ga_ulong)0;
    for (ga_uint b = 0; b < bits; b++) {
      const bool one = (d >> b) & 1;
      const ga_ulong with = __builtin_amdgcn_ballot_w64(one);
      peers &= one ? with : ~with;
    }
    const ga_uint before = __builtin_amdgcn_mbcnt_hi((ga_uint)(peers >> 32), __builtin_amdgcn_mbcnt_lo((ga_uint)peers, 0));
    const ga_uint have = counts[wave][d];
    rank[r] = have + before;
    __builtin_amdgcn_wave_barrier();
    if (before == 0) counts[wave][d] = (ga_ushort)(have + (ga_uint)__builtin_popcountll(peers));
    __builtin_amdgcn_wave_barrier();
  }
  local_barrier();
}
/* counts[wave][digit] becomes what the earlier wavefronts have of the digit; returns, in
 * lane b, how many of digit b the group has */
LM_FN ga_uint lm_wave_prefix(volatile ga_ushort (*counts)[LM_BINS], ga_uint bits) {
  ga_uint total = 0;
  if (LID_0 < (1u << bits)) {
    for (int w = 0; w < 16; w++) {
      const ga_uint c = counts[w][LID_0];
      counts[w][LID_0] = (ga_ushort)total;
      total += c;
    }
  }
  return total;
}

/* Up to 1024 * LM_R tokens: group 0 sorts them by itself, in its LDS. */
KERNEL void __launch_bounds__(1024) lm_sort_small(const lm_sorting p) {
  if (GID_0 != 0) {
    lm_clear(p, 1);
    return;
  }
  LOCAL_MEM ga_ushort counts[16][LM_BINS] __attribute__((aligned(16)));
  LOCAL_MEM ga_uint keys[1024 * LM_R];
  LOCAL_MEM ga_ushort places[1024 * LM_R];
  const ga_uint first = (LID_0 >> 6) * 64 * LM_R + (LID_0 & 63);
  ga_uint k[LM_R], at[LM_R], rank[LM_R];
#pragma unroll
  for (int r = 0; r < LM_R; r++) {
    at[r] = first + r * 64;
    k[r] = at[r] < p.n ? lm_first_key(p, at[r]) : 0xffffffffu;
  }
  for (ga_uint pass = 0; pass < p.passes; pass++) {
    const ga_uint shift = pass * p.bits, mask = (1u << p.bits) - 1;
    lm_rank(k, rank, counts, shift, p.bits);
    const ga_uint total = lm_wave_prefix(counts, p.bits);
    const ga_uint base = lm_scan(total);
    if (LID_0 < (1u << p.bits))
      for (int w = 0; w < 16; w++) counts[w][LID_0] = (ga_ushort)(counts[w][LID_0] + base);
    local_barrier();
#pragma unroll
    for (int r = 0; r < LM_R; r++) {
      const ga_uint to = counts[LID_0 >> 6][(k[r] >> shift) & mask] + rank[r];
      keys[to] = k[r];
      places[to] = (ga_ushort)at[r];
    }
    local_barrier();
#pragma unroll
    for (int r = 0; r < LM_R; r++) {
      k[r] = keys[first + r * 64];
      at[r] = places[first + r * 64];
    }
    local_barrier();
  }
#pragma unroll
  for (int r = 0; r < LM_R; r++) {
    const ga_uint i = first + r * 64;
    if (i < p.n) {
      p.key[i] = k[r];
      p.order[i] = at[r];
    }
  }
}

/* More tokens: a pass is three launches.  What every group has of each digit; */
KERNEL void __launch_bounds__(1024) lm_sort_count(const lm_sorting p) {
  if (GID_0 >= p.groups) {
    lm_clear(p, p.groups);
    return;
  }
  LOCAL_MEM ga_uint bins[LM_BINS];
  bins[LID_0] = 0;
  local_barrier();
  const ga_uint first = GID_0 * 1024 * LM_R + LID_0;
#pragma unroll
  for (int r = 0; r < LM_R; r++) {
    const ga_uint i = first + r * 1024;
    if (i < p.n) {
      const ga_uint k = p.shift == 0 ? lm_first_key(p, i) : p.key_in[i];
      atomicAdd(&bins[(k >> p.shift) & ((1u << p.bits) - 1)], 1u);
    }
  }
  local_barrier();
  if (LID_0 < (1u << p.bits)) p.counts[p.direct ? (GID_0 << p.bits) + LID_0 : (ga_size)LID_0 * p.groups + GID_0] = bins[LID_0];
}
/* what the earlier groups have of a digit, a wavefront per digit; */
KERNEL void __launch_bounds__(1024) lm_sort_scan(const lm_sorting p) {
  const ga_uint busy = ((1u << p.bits) + 15) / 16;
  if (GID_0 >= busy) {
    lm_clear(p, busy);
    return;
  }
  const ga_uint digit = GID_0 * 16 + (LID_0 >> 6), lane = LID_0 & 63;
  if (digit >= (1u << p.bits)) return;
  GLOBAL_MEM ga_uint *c = p.counts + (ga_size)digit * p.groups;
  ga_uint before = 0;
  for (ga_uint base = 0; base < p.groups; base += 64) {
    const ga_uint x = base + lane < p.groups ? c[base + lane] : 0;
    ga_uint s = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const ga_uint y = (ga_uint)__builtin_amdgcn_ds_bpermute((int)((lane - d) << 2), (int)s);
      if (lane >= d) s += y;
    }
    if (base + lane < p.groups) c[base + lane] = before + s - x;
    before += (ga_uint)__builtin_amdgcn_readlane((int)s, 63);
  }
  if (lane == 0) p.counts[((ga_size)p.groups << p.bits) + digit] = before;
}
/* every token to its place. */
KERNEL void __launch_bounds__(1024) lm_sort_move(const lm_sorting p) {
  if (GID_0 >= p.groups) {
    lm_clear(p, p.groups);
    return;
  }
  LOCAL_MEM ga_ushort counts[16][LM_BINS] __attribute__((aligned(16)));
  LOCAL_MEM ga_uint base[LM_BINS];
  const ga_uint first = GID_0 * 1024 * LM_R + (LID_0 >> 6) * 64 * LM_R + (LID_0 & 63);
  ga_uint k[LM_R], rank[LM_R];
#pragma unroll
  for (int r = 0; r < LM_R; r++) {
    const ga_uint i = first + r * 64;
    k[r] = i < p.n ? (p.shift == 0 ? lm_first_key(p, i) : p.key_in[i]) : 0xffffffffu;
  }
  lm_rank(k, rank, counts, p.shift, p.bits);
  (void)lm_wave_prefix(counts, p.bits);
  const bool mine = LID_0 < (1u << p.bits);
  ga_uint total = 0, before = 0;   /* of digit LID_0 in all groups, and in the earlier ones */
  if (!p.direct) {
    if (mine) total = p.counts[((ga_size)p.groups << p.bits) + LID_0], before = p.counts[(ga_size)LID_0 * p.groups + GID_0];
  } else if (mine) {
#pragma unroll 16
    for (ga_uint g = 0; g < p.groups; g++) {
      const ga_uint c = p.counts[(g << p.bits) + LID_0];
      total += c;
      before += g < GID_0 ? c : 0;
    }
  }
  const ga_uint start = lm_scan(total);
  if (mine) base[LID_0] = start + before;
  local_barrier();
#pragma unroll
  for (int r = 0; r < LM_R; r++) {
    const ga_uint i = first + r * 64, d = (k[r] >> p.shift) & ((1u << p.bits) - 1);
    if (i < p.n) {
      const ga_uint to = base[d] + counts[LID_0 >> 6][d] + rank[r];
      p.key[to] = k[r];
      p.order[to] = p.shift == 0 ? i : p.order_in[i];
    }
  }
}
#endif

#if LM_KIND == LM_K_EMBED_GRAD
/* columns of a lane: 16 bytes of the wider side, so that either side's accesses are whole lines */
#define LM_W (sizeof(LM_X) > sizeof(LM_O) ? 16 / (int)sizeof(LM_X) : 16 / (int)sizeof(LM_O))
struct lm_embed_grad {
  GLOBAL_MEM LM_O *grad;
  GLOBAL_MEM const LM_X *dout;
  GLOBAL_MEM const ga_uint *key, *order;   /* the sorted tokens */
  GLOBAL_MEM float *partials;              /* [chunk][2][tiles * 64 * LM_W] */
  GLOBAL_MEM const LM_ID *ids;             /* of few tokens */
  GLOBAL_MEM ga_int *err;
  ga_long id_step, ignore;
  ga_long grad_row, dout_row, v, d;
  float scale;
  ga_int accumulate;
  ga_uint n, chunk, chunks, tiles, rows, lanes_log2;
  ga_uint dense, part_tiles;                   /* the table's rows lie end to end */
};

/* The columns of a lane: LM_W from `from` on, of which the first `skip` belong
 * to the lane before it (at a row's end, where the last LM_W columns are
 * fetched), and `cols` are inside the row. */
struct lm_columns {
  ga_long from;
  ga_int skip, cols;
};
LM_FN lm_columns lm_columns_of(ga_long col, ga_long d) {
  lm_columns c = {col, 0, LM_W};
  if (d < LM_W) {
    c.cols = col == 0 ? (ga_int)d : 0;
    c.from = 0;
  } else if (d - col < LM_W) {
    c.from = d - LM_W;
    c.skip = col >= d ? LM_W : (ga_int)(col - c.from);
  }
  return c;
}

/* One run's sum is complete. */
LM_FN void lm_write_run(const lm_embed_grad &p, ga_uint key, const lm_columns &c, const float (&sum)[LM_W]) {
  GLOBAL_MEM LM_O *g = lm_at(p.grad, (ga_long)key * p.grad_row) + c.from;
  float y[LM_W];
#pragma unroll
  for (int e = 0; e < LM_W; e++) y[e] = p.scale * sum[e];
  if (c.skip == 0 && c.cols == LM_W) {
    if (p.accumulate) {
      float have[LM_W];
      lm_load(g, have);
#pragma unroll
      for (int e = 0; e < LM_W; e++) y[e] += have[e];
    }
    lm_store(g, y);
  } else {
#pragma unroll
    for (int e = 0; e < LM_W; e++)
      if (e >= c.skip && e < c.cols) lm_put(g + e, p.accumulate ? lm_get(g[e]) + y[e] : y[e]);
  }
}

#define LM_AHEAD 8   /* rows in flight */
/* the columns of rows at[..] of dout; unconditional loads: all of them in flight */
LM_FN void lm_fetch_rows(const lm_embed_grad &p, const ga_uint (&at)[LM_AHEAD], const lm_columns &c, float (&y)[LM_AHEAD][LM_W]) {
  if (p.d >= LM_W) {
#pragma unroll
    for (int u = 0; u < LM_AHEAD; u++) lm_load(lm_at(p.dout, (ga_long)at[u] * p.dout_row) + c.from, y[u]);
  } else {
#pragma unroll
    for (int u = 0; u < LM_AHEAD; u++)
#pragma unroll
      for (int e = 0; e < LM_W; e++) y[u][e] = e < c.cols ? (float)lm_get(lm_at(p.dout, (ga_long)at[u] * p.dout_row)[e]) : 0.0f;
  }
}

/* Few tokens need no sorting: a group takes p.rows rows of the table and up to
 * four times 64 * LM_W columns of them, zeroes them, end to end if it can, and
 * looks all ids through once, which leaves a mask of the tokens of each row; it
 * adds those in order and writes the rows that have some.  One launch in place of four. */
#define LM_FEW 256        /* tokens at most */
#define LM_FEW_ROWS 512   /* rows at most */
/* A wavefront adds the tokens of a row, those whose bits are set, over one tile of columns. */
LM_FN void lm_add_few(const lm_embed_grad &p, ga_uint key, ga_uint tile, ga_ulong (&left)[LM_FEW / 64]) {
  const ga_uint lane = LID_0 & 63;
  const lm_columns mine = lm_columns_of(((ga_long)tile * 64 + lane) * LM_W, p.d);
  float sum[LM_W];
#pragma unroll
  for (int e = 0; e < LM_W; e++) sum[e] = 0.0f;
#pragma unroll
  for (int w = 0; w < LM_FEW / 64; w++) {
    while (left[w] != 0) {
      ga_uint at[LM_AHEAD];
      ga_uint n = 0;
#pragma unroll
      for (int u = 0; u < LM_AHEAD; u++) {
        at[u] = left[w] != 0 ? w * 64 + (ga_uint)__builtin_ctzll(left[w]) : at[u > 0 ? u - 1 : 0];
        n += left[w] != 0;
        left[w] &= left[w] - 1;
      }
      float y[LM_AHEAD][LM_W];
      lm_fetch_rows(p, at, mine, y);
#pragma unroll
      for (int u = 0; u < LM_AHEAD; u++) {
        if (u < n) {
#pragma unroll
          for (int e = 0; e < LM_W; e++) sum[e] += y[u][e];
        }
      }
    }
  }
  lm_write_run(p, key, mine, sum);
}
/* What is added to: a group for each token and p.part_tiles tiles, one tile a
 * wavefront at a time; the first token of a row adds them all. */
LM_FN void lm_add_to_few(const lm_embed_grad &p, ga_long id) {
  LOCAL_MEM ga_long ids[LM_FEW];
  LOCAL_MEM ga_ulong mask[LM_FEW / 64];
  const ga_uint parts = (p.tiles + p.part_tiles - 1) / p.part_tiles, token = GID_0 / parts, part = GID_0 % parts;
  ids[LID_0] = id;
  local_barrier();
  const ga_long mine = ids[token];
  const ga_ulong m = __builtin_amdgcn_ballot_w64(id == mine);
  if ((LID_0 & 63) == 0) mask[LID_0 >> 6] = m;
  local_barrier();
  if (mine < 0) return;
  ga_ulong all[LM_FEW / 64];
#pragma unroll
  for (int w = LM_FEW / 64 - 1; w >= 0; w--) {
    all[w] = mask[w];
    all[w] = (ga_ulong)(ga_uint)__builtin_amdgcn_readfirstlane((int)(all[w] >> 32)) << 32 |
             (ga_uint)__builtin_amdgcn_readfirstlane((int)all[w]);
    if (w == token >> 6 ? (all[w] & ((1ull << (token & 63)) - 1)) != 0 : w < token >> 6 && all[w] != 0) return;
  }
  for (ga_uint i = LID_0 >> 6; i < p.part_tiles && part * p.part_tiles + i < p.tiles; i += 4) {
    ga_ulong left[LM_FEW / 64];
#pragma unroll
    for (int w = 0; w < LM_FEW / 64; w++) left[w] = all[w];
    lm_add_few(p, (ga_uint)mine, part * p.part_tiles + i, left);
  }
}
KERNEL void __launch_bounds__(256) lm_embed_grad_few(const lm_embed_grad p) {
  LOCAL_MEM ga_ulong masks[LM_FEW_ROWS][LM_FEW / 64];
  LOCAL_MEM ga_ushort with[LM_FEW];
  LOCAL_MEM ga_uint count;
  LOCAL_MEM ga_uint some, next;   /* do these rows, does the one after them have tokens */
  const ga_uint lane = LID_0 & 63, wave = LID_0 >> 6;
  const ga_uint parts = (p.tiles + p.part_tiles - 1) / p.part_tiles, part = GID_0 % parts, tile0 = part * p.part_tiles;
  const ga_uint tiles = p.tiles - tile0 < p.part_tiles ? p.tiles - tile0 : p.part_tiles;
  const ga_long r0 = (ga_long)(GID_0 / parts) * p.rows;
  const ga_uint rows = r0 >= p.v ? 0 : p.v - r0 < p.rows ? (ga_uint)(p.v - r0) : p.rows;
  const ga_long id = LID_0 < p.n ? lm_id(*lm_at(p.ids, (ga_long)LID_0 * p.id_step), p.ignore, LM_NONE, p.v) : -1;
  if (id == -2) *p.err = -1;
  if (p.accumulate) {
    lm_add_to_few(p, id);
    return;
  }
  if (LID_0 == 0) some = next = count = 0;
  for (ga_uint i = LID_0; i < rows * (LM_FEW / 64); i += 256) (&masks[0][0])[i] = 0;
  GLOBAL_MEM char *b = (GLOBAL_MEM char *)p.grad + r0 * p.grad_row;
  const ga_long row = p.d * (ga_long)sizeof(LM_O);
  const bool flat = p.dense && parts == 1, shared = flat && row >= 16 && (row & 15) != 0;
  if (rows > 0 && !shared) {
    if (flat) {
      lm_zero(b, rows * row, LID_0, 256);
    } else {
      const ga_long col = (ga_long)tile0 * 64 * LM_W, cols = p.d - col < tiles * 64 * LM_W ? p.d - col : tiles * 64 * LM_W;
      for (ga_uint k = 0; k < rows; k++)
        lm_zero(b + k * p.grad_row + col * (ga_long)sizeof(LM_O), cols * (ga_long)sizeof(LM_O), LID_0, 256);
    }
  }
  local_barrier();
  if (id >= r0 && id < r0 + rows) {
    atomicOr((unsigned long long *)&masks[id - r0][wave], 1ull << lane);
    some = 1;
  }
  if (id == r0 + rows) next = 1;
  local_barrier();
  if (shared) {
    /* A 16-byte chunk that two groups share is one store of the first of them,
     * but where the second one's first row has tokens, and so is not all zeros
     * (22723 rows of 4413 bfloat16 42 us, with stores of what is left at both ends 48). */
    ga_long from = 0, to = rows * row;
    if (r0 > 0 && (masks[0][0] | masks[0][1] | masks[0][2] | masks[0][3]) == 0) from = (ga_long)(-(ga_size)b & 15);
    if (r0 + rows < p.v && !next) to += (ga_long)(-(ga_size)(b + to) & 15);
    lm_zero(b + from, to - from, LID_0, 256);
  }
  if (!some) return;
  for (ga_uint k = LID_0; k < rows; k += 256)    /* (in any order: each row is a sum of its own) */
    if (masks[k][0] | masks[k][1] | masks[k][2] | masks[k][3]) with[atomicAdd(&count, 1u)] = (ga_ushort)k;
  /* (the zeros are in the L2 before a sum follows them) */
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  local_barrier();
  for (ga_uint unit = wave; unit < count * tiles; unit += 4) {
    const ga_uint k = (ga_uint)__builtin_amdgcn_readfirstlane((int)with[unit / tiles]), tile = tile0 + unit % tiles;
    ga_ulong left[LM_FEW / 64];
#pragma unroll
    for (int w = 0; w < LM_FEW / 64; w++) {
      left[w] = masks[k][w];
      left[w] = (ga_ulong)(ga_uint)__builtin_amdgcn_readfirstlane((int)(left[w] >> 32)) << 32 |
                (ga_uint)__builtin_amdgcn_readfirstlane((int)left[w]);
    }
    lm_add_few(p, (ga_uint)(r0 + k), tile, left);
  }
}

/* A wavefront adds the rows of a chunk of the sorted tokens, in their order, over
 * 64 * LM_W columns.  A run of equal ids that lies inside the chunk is written
 * when it ends; what a chunk has of a run that began earlier (slot 0), or that
 * goes on in the next (slot 1), is left for lm_embed_grad_join.  No atomics: what a row's sum
 * consists of, and in which order, is the same on every call.  Bound by memory, and by how
 * evenly the wavefronts' work falls out: 65536 tokens of 2048 bfloat16, 0.3 of them none, added to
 * floats 95 us (0.42 GB, 4.4 TB/s); more rows in flight than 8 were no faster. */
#if LM_NARROW
/* Short rows: 2^lanes_log2 lanes have a chunk, several chunks lie side by side in
 * a wavefront, and what is uniform in a wavefront with one chunk is so here
 * among the lanes of each. */
#define LM_FROM(x, i) ((ga_uint)__builtin_amdgcn_ds_bpermute((int)((first + (i)) << 2), (int)(x)))
#else
#define LM_FROM(x, i) ((ga_uint)__builtin_amdgcn_readlane((int)(x), (int)(i)))
#endif
KERNEL void __launch_bounds__(256) lm_embed_grad_sum(const lm_embed_grad p) {
#if LM_NARROW
  const ga_uint lanes = 1u << p.lanes_log2;
  const ga_uint lane = LID_0 & (lanes - 1), first = (LID_0 & 63) - lane;
  const ga_uint chunk = (GID_0 * 256 + LID_0) >> p.lanes_log2, tile = 0;
#else
  const ga_uint lanes = 64;
  const ga_uint unit = (ga_uint)__builtin_amdgcn_readfirstlane((int)(GID_0 * 4 + (LID_0 >> 6)));
  const ga_uint chunk = unit / p.tiles, tile = unit % p.tiles, lane = LID_0 & 63;
#endif
  if (chunk >= p.chunks) return;
  const ga_uint p0 = chunk * p.chunk;
  const ga_uint n = p.n - p0 < p.chunk ? p.n - p0 : p.chunk;
  const ga_long col = ((ga_long)tile * 64 + lane) * LM_W;
  const lm_columns mine = lm_columns_of(col, p.d);
  const ga_uint none = (ga_uint)p.v;
  GLOBAL_MEM float *slots = p.partials + (ga_size)chunk * 2 * p.tiles * 64 * LM_W + col;
  float sum[LM_W];
#pragma unroll
  for (int e = 0; e < LM_W; e++) sum[e] = 0.0f;
  const auto leave = [&](int slot) {
#pragma unroll
    for (int e = 0; e < LM_W; e++) slots[(ga_size)slot * p.tiles * 64 * LM_W + e] = sum[e];
  };
  const ga_uint before = p0 > 0 ? p.key[p0 - 1] : 0xffffffffu;
  const ga_uint after = p0 + n < p.n ? p.key[p0 + n] : 0xffffffffu;
  ga_uint run = p.key[p0];
  if (run == none) return;     /* no tokens, to the end */
  bool here = run != before;   /* the run began in this chunk */
  for (ga_uint sub = 0; sub < n; sub += lanes) {
    const ga_uint i = p0 + sub + lane;
    const bool in = sub + lane < n;
    const ga_uint keys = in ? p.key[i] : none, places = in ? p.order[i] : 0;
    const ga_uint m = n - sub < lanes ? n - sub : lanes;
    for (ga_uint j = 0; j < m; j += LM_AHEAD) {
      float y[LM_AHEAD][LM_W];
      ga_uint k[LM_AHEAD], at[LM_AHEAD];
#pragma unroll
      for (int u = 0; u < LM_AHEAD; u++) {     /* (past m: the last one once more) */
        const ga_uint w = j + u < m ? j + u : m - 1;
        k[u] = LM_FROM(keys, w);
        at[u] = LM_FROM(places, w);
      }
      lm_fetch_rows(p, at, mine, y);
#pragma unroll
      for (int u = 0; u < LM_AHEAD; u++) {
        if (j + u >= m) continue;
        if (k[u] != run) {
          if (here) lm_write_run(p, run, mine, sum);
          else leave(0);
#pragma unroll
          for (int e = 0; e < LM_W; e++) sum[e] = 0.0f;
          run = k[u];
          here = true;
        }
        if (k[u] != none) {
#pragma unroll
          for (int e = 0; e < LM_W; e++) sum[e] += y[u][e];
        }
      }
    }
  }
  if (run == none) return;
  if (here && run != after) lm_write_run(p, run, mine, sum);
  else leave(here ? 1 : 0);
}

/* The runs that cross chunks: the group of the chunk where a run begins adds
 * its parts.  A long run's parts are split over as many sets of lanes as the
 * group has for the columns, which meet in the LDS in fixed order (after the sums above 9 us). */
KERNEL void __launch_bounds__(256) lm_embed_grad_join(const lm_embed_grad p) {
  const ga_uint chunk = GID_0 / p.tiles, tile = GID_0 % p.tiles;
#if LM_NARROW
  const ga_uint lanes_log2 = p.lanes_log2;
#else
  const ga_uint lanes_log2 = 6;
#endif
  const ga_uint lane = LID_0 & ((1u << lanes_log2) - 1), set = LID_0 >> lanes_log2, sets = 256u >> lanes_log2;
  const ga_uint p0 = chunk * p.chunk;
  if (p0 + p.chunk >= p.n) return;             /* the last chunk: nothing goes on */
  const ga_uint run = p.key[p0 + p.chunk];
  if (run == (ga_uint)p.v || p.key[p0 + p.chunk - 1] != run) return;
  if (p0 > 0 && p.key[p0 - 1] == run) return;  /* it began earlier */
  /* the chunks after this one that begin inside the run */
  ga_uint parts = 0;
  for (;;) {
    const ga_ulong at = (ga_ulong)(chunk + 1 + parts + (LID_0 & 63)) * p.chunk;
    const ga_ulong in = __builtin_amdgcn_ballot_w64(at < p.n && p.key[at < p.n ? at : 0] == run);
    if (~in == 0) {
      parts += 64;
      continue;
    }
    parts += (ga_uint)__builtin_ctzll(~in);
    break;
  }
  const ga_long col = ((ga_long)tile * 64 + lane) * LM_W;
  const ga_size pitch = (ga_size)p.tiles * 64 * LM_W;
  GLOBAL_MEM const float *next = p.partials + (ga_size)(chunk + 1) * 2 * pitch + col;
  const bool split = parts > 4;
  const ga_uint share = split ? (parts + sets - 1) / sets : parts;
  const ga_uint from = set * share < parts ? set * share : parts, to = from + share < parts ? from + share : parts;
  float sum[LM_W];
#pragma unroll
  for (int e = 0; e < LM_W; e++) sum[e] = set == 0 ? next[e - (ga_long)pitch] : 0.0f;
#pragma unroll 8
  for (ga_uint i = from; i < to; i++) {
#pragma unroll
    for (int e = 0; e < LM_W; e++) sum[e] += next[(ga_size)i * 2 * pitch + e];
  }
  if (split) {
    LOCAL_MEM float meet[256][LM_W];
#pragma unroll
    for (int e = 0; e < LM_W; e++) meet[LID_0][e] = sum[e];
    local_barrier();
    if (set == 0) {
      for (ga_uint w = 1; w < sets; w++)
#pragma unroll
        for (int e = 0; e < LM_W; e++) sum[e] += meet[(w << lanes_log2) + lane][e];
    }
  }
  if (set == 0) lm_write_run(p, run, lm_columns_of(col, p.d), sum);
}
#endif

/* R = by * m, the largest logit in powers of two, is rounded to a float, and what the rounding leaves,
 * r = by * m - R, is part of every exponent by * x - R: of the largest element's too, which is r in place of 0.
 * Below 2^30 that is 32 at most, half a step of R, and the exponential and the sums hold it. From there on r would
 * leave the range of the exponential (past 2^31: 128 and more); but by * x of neighbouring numbers is 64 or more apart
 * then, 2^-64 of an element is none, and so only the elements that are equal to m count, with exponent 0. */
#define LM_FAR 1073741824.0f

#if LM_KIND == LM_K_LOGPROBS
struct lm_logprobs {
  GLOBAL_MEM const LM_X *logits;
  GLOBAL_MEM const LM_ID *ids;   /* NULL: no logp */
  GLOBAL_MEM float *logp, *entropy, *stats, *top_logp;   /* NULL: not wanted */
  GLOBAL_MEM void *top_ids;
  GLOBAL_MEM ga_int *err;
  GLOBAL_MEM char *partials;     /* of rows in pieces: lm_state, then the alternatives' keys */
  ga_long row, id_step, logp_step, entropy_step, stats_row, stats_col;
  ga_long topl_row, topl_col, topi_row, topi_col;
  ga_long t, v, ignore;
  float scale, by;               /* by = scale * log2(e) */
  ga_int top, top_long;
  ga_uint pieces, piece_chunks, partial_bytes;
  ga_uint pad;
  GLOBAL_MEM ga_uint *counters;  /* one zero per row in pieces */
};

/* Softmax statistics of some elements x of a row.  With R(m) = by * m, rounded,
 *   s = sum of 2^(by * x - R(m)),   w = sum of (by * x - R(m)) 2^(by * x - R(m)),
 * where m is the largest x; R(m) being a number that is known exactly, its
 * rounding is no error of s or w.  One multiply-add and one exponential per
 * element.  -inf has no part in either sum.  Where |R| is past LM_FAR s
 * counts the elements that are equal to m, and w is 0: rows of a mask's value, and
 * what a lane has of one before it meets anything else. */
struct lm_state {
  float m, s, w, pad;
};
#define LM_LOWEST (-3.402823466e+38f)

/* R(from) - R(to), from <= to, R(to) no farther out than LM_FAR; at least -300, which is as good as -inf for the
 * exponential and safe to multiply with 0 */
LM_FN float lm_near_shift(float from, float to, float by) {
  const float d = __builtin_fmaxf(from * by - to * by, -300.0f);
  return from == to ? 0.0f : d;
}
/* the same for any; farther out numbers that differ may have one R, and none but equal ones count */
LM_FN float lm_shift(float from, float to, float by) {
  const float r = to * by, d = __builtin_fabsf(r) <= LM_FAR ? __builtin_fmaxf(from * by - r, -300.0f) : -300.0f;
  return from == to ? 0.0f : d;
}
LM_FN void lm_rescale(lm_state &a, float m, float d) {   /* d: the shift from a.m to m */
  const float f = __builtin_amdgcn_exp2f(d);
#if LM_ENT
  a.w = f * __builtin_fmaf(a.s, d, a.w);
#endif
  a.s *= f;
  a.m = m;
}
LM_FN void lm_join(lm_state &a, lm_state b, float by) {
  const float m = __builtin_fmaxf(a.m, b.m);
  lm_rescale(a, m, lm_shift(a.m, m, by));
  lm_rescale(b, m, lm_shift(b.m, m, by));
  a.s += b.s;
  a.w += b.w;
}
template <int MASK> LM_FN void lm_max_xor(float &m) { m = __builtin_fmaxf(m, lm_xor<MASK>(m)); }
template <int MASK> LM_FN void lm_sum_xor(lm_state &a) {
  a.s += lm_xor<MASK>(a.s);
#if LM_ENT
  a.w += lm_xor<MASK>(a.w);
#endif
}
/* The maximum first, so that a lane rescales once. */
LM_FN void lm_join_wave(lm_state &a, float by) {
  float m = a.m;
  lm_max_xor<1>(m); lm_max_xor<2>(m); lm_max_xor<7>(m); lm_max_xor<15>(m); lm_max_xor<16>(m); lm_max_xor<32>(m);
  lm_rescale(a, m, lm_shift(a.m, m, by));
  lm_sum_xor<1>(a); lm_sum_xor<2>(a); lm_sum_xor<7>(a); lm_sum_xor<15>(a); lm_sum_xor<16>(a); lm_sum_xor<32>(a);
}
LM_FN float lm_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
/* the largest of y[0..N) and a */
template <int N> LM_FN float lm_max_of(const float (&y)[N], float a) {
#pragma unroll
  for (int i = 0; i + 1 < N; i += 2) a = lm_max3(a, y[i], y[i + 1]);
  if (N & 1) a = __builtin_fmaxf(a, y[N - 1]);
  return a;
}

/* N elements of every lane join its statistics. */
template <int N> LM_FN void lm_add(lm_state &a, const float (&y)[N], float most, float by) {
  const float m = __builtin_fmaxf(a.m, most), r = m * by;
  const bool far = !(__builtin_fabsf(r) <= LM_FAR);
  float s[2] = {0.0f, 0.0f}, w[2] = {0.0f, 0.0f};
  if (__builtin_amdgcn_ballot_w64(far) == 0) {
    lm_rescale(a, m, lm_near_shift(a.m, m, by));
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float t = __builtin_fmaf(y[i], by, -r), e = __builtin_amdgcn_exp2f(t);
      s[i & 1] += e;
#if LM_ENT
      w[i & 1] = __builtin_fmaf(e, t, w[i & 1]);
#endif
    }
#if LM_ENT
    /* 0 * -inf: some element is -inf.  Once more, with products that stay finite. */
    if (__builtin_amdgcn_ballot_w64(w[0] + w[1] != w[0] + w[1]) != 0) {
      w[0] = w[1] = 0.0f;
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float t = __builtin_fmaf(y[i], by, -r), e = __builtin_amdgcn_exp2f(t);
        w[i & 1] = __builtin_fmaf(e, __builtin_fmaxf(t, -300.0f), w[i & 1]);
      }
    }
#endif
  } else {
    lm_rescale(a, m, lm_shift(a.m, m, by));
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float t = far ? 0.0f : __builtin_fmaf(y[i], by, -r);
      float e = __builtin_amdgcn_exp2f(t);
      if (far) e = y[i] == m ? 1.0f : (y[i] != y[i] ? y[i] : 0.0f);
      s[i & 1] += e;
      w[i & 1] = __builtin_fmaf(e, __builtin_fmaxf(t, -300.0f), w[i & 1]);
    }
  }
  a.s += s[0] + s[1];
#if LM_ENT
  a.w += w[0] + w[1];
#endif
}

/* ---- the alternatives -----------------------------------------------------------
 * A wavefront keeps its best 64 elements as keys, sorted, one per lane: the
 * upper 32 of a key's 62 bits order the values (-0 as 0), the lower 30 prefer
 * low indices; 0 is no element.  Keys of 62 bits are ordered as the doubles below 2 that
 * have these bits, so that a comparison and its two outcomes are the maximum
 * and the minimum of two doubles, with no way through a scalar mask.
 * -inf is never kept: what is missing in the end is filled up by a look at the row. */
#define LM_INDEX 0x3fffffffu
LM_FN ga_ulong lm_key(float y, ga_uint index) {
  const ga_uint b = __builtin_bit_cast(ga_uint, y + 0.0f);
  const ga_uint o = b ^ ((ga_uint)((ga_int)b >> 31) | 0x80000000u);
  return (ga_ulong)(o >> 2) << 32 | (o << 30 | (LM_INDEX - index));
}
LM_FN float lm_key_value(ga_ulong k) {
  const ga_uint b = (ga_uint)(k >> 30);
  return __builtin_bit_cast(float, b ^ ((b & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}
LM_FN ga_uint lm_key_index(ga_ulong k) { return LM_INDEX - ((ga_uint)k & LM_INDEX); }
LM_FN ga_ulong lm_larger(ga_ulong a, ga_ulong b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(__builtin_bit_cast(double, a)), "v"(__builtin_bit_cast(double, b)));
  return __builtin_bit_cast(ga_ulong, r);
}
LM_FN ga_ulong lm_smaller(ga_ulong a, ga_ulong b) {
  double r;
  asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(__builtin_bit_cast(double, a)), "v"(__builtin_bit_cast(double, b)));
  return __builtin_bit_cast(ga_ulong, r);
}

/* one step of a sorting network: of lane and lane ^ MASK the lower one keeps the larger key */
template <int MASK> LM_FN void lm_step(ga_ulong &k) {
  const ga_ulong other = lm_xor<MASK>(k);
  const ga_uint top_bit = 1u << (31 - __builtin_clz(MASK));
  const bool lower = (LID_0 & top_bit) == 0;
  const ga_ulong l = lm_larger(k, other), s = lm_smaller(k, other);
  k = lower ? l : s;
}
LM_FN void lm_sort(ga_ulong &k) {   /* descending over the 64 lanes */
  lm_step<1>(k);
  lm_step<3>(k); lm_step<1>(k);
  lm_step<7>(k); lm_step<2>(k); lm_step<1>(k);
  lm_step<15>(k); lm_step<4>(k); lm_step<2>(k); lm_step<1>(k);
  lm_step<31>(k); lm_step<8>(k); lm_step<4>(k); lm_step<2>(k); lm_step<1>(k);
  lm_step<63>(k); lm_step<16>(k); lm_step<8>(k); lm_step<4>(k); lm_step<2>(k); lm_step<1>(k);
}
/* list := the best 64 of two sorted lists, sorted */
LM_FN void lm_merge(ga_ulong &list, ga_ulong other) {
  const ga_ulong r = lm_xor<63>(other);
  list = lm_larger(list, r);
  lm_step<32>(list); lm_step<16>(list); lm_step<8>(list); lm_step<4>(list); lm_step<2>(list); lm_step<1>(list);
}
LM_FN ga_ulong lm_lane(ga_ulong k, int lane) {
  return (ga_ulong)(ga_uint)__builtin_amdgcn_readlane((int)(ga_uint)(k >> 32), lane) << 32 |
         (ga_uint)__builtin_amdgcn_readlane((int)(ga_uint)k, lane);
}

/* The same network on 32-bit words: a word that n of the 64 are not below, for every
 * lane; the n-th largest, or, for n up to 8, the n-th largest of the 16 maxima of four
 * lanes, which costs half as much and lets few more pass (for 5 of 64 5.7 in place of 5.2). */
template <int MASK> LM_FN void lm_step32(ga_uint &k) {
  const ga_uint other = lm_xor<MASK>(k);
  const bool lower = (LID_0 & (1u << (31 - __builtin_clz(MASK)))) == 0;
  k = lower ? max(k, other) : min(k, other);
}
LM_FN ga_uint lm_kth(ga_uint k, ga_int n) {
  if (n <= 8) {
    k = max(k, lm_xor<16>(k));
    k = max(k, lm_xor<32>(k));
  }
  lm_step32<1>(k);
  lm_step32<3>(k); lm_step32<1>(k);
  lm_step32<7>(k); lm_step32<2>(k); lm_step32<1>(k);
  lm_step32<15>(k); lm_step32<4>(k); lm_step32<2>(k); lm_step32<1>(k);
  if (n > 8) {
    lm_step32<31>(k); lm_step32<8>(k); lm_step32<4>(k); lm_step32<2>(k); lm_step32<1>(k);
    lm_step32<63>(k); lm_step32<16>(k); lm_step32<8>(k); lm_step32<4>(k); lm_step32<2>(k); lm_step32<1>(k);
  }
  return (ga_uint)__builtin_amdgcn_readlane((int)k, n - 1);
}

/* A wavefront's best elements: a sorted list, and `n` that wait to join it, one
 * per lane in no order.  An element that is not above `bar`, or equal to it at
 * an index below bar_index, is none of the `top` best. */
struct lm_best {
  ga_ulong list, waiting;
  ga_uint n, bar_index;
  float bar;
};
LM_FN float lm_uniform(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
LM_FN void lm_settle(lm_best &b, ga_int top) {
  if (b.n == 0) return;
  const ga_uint lane = LID_0 & 63;
  if (b.n <= 16) {
    /* a few: every lane counts the keys above its own, and sends its key to that place */
    ga_uint place = lane;
    if (lane < b.n) place = 0;
    for (ga_uint i = 0; i < b.n; i++) {
      const ga_ulong k = lm_lane(b.waiting, (int)i);
      place += lane < b.n && k > b.waiting;
    }
    const ga_uint lo = (ga_uint)__builtin_amdgcn_ds_permute((int)(place << 2), (int)(ga_uint)b.waiting);
    const ga_uint hi = (ga_uint)__builtin_amdgcn_ds_permute((int)(place << 2), (int)(ga_uint)(b.waiting >> 32));
    b.waiting = (ga_ulong)hi << 32 | lo;
  } else {
    lm_sort(b.waiting);
  }
  if (__builtin_amdgcn_ballot_w64(b.list != 0) == 0) b.list = b.waiting;
  else lm_merge(b.list, b.waiting);
  b.waiting = 0;
  b.n = 0;
  const ga_ulong k = lm_lane(b.list, top - 1);
  if (k != 0) {
    b.bar = lm_uniform(lm_key_value(k));
    b.bar_index = lm_key_index(k);
  }
}
LM_FN ga_uint lm_ordered(float y) { return (ga_uint)(lm_key(y, 0) >> 30); }
LM_FN void lm_raise(lm_best &b, ga_uint ordered) {
  const float t = lm_uniform(lm_key_value((ga_ulong)ordered << 30));
  if (t > b.bar) {
    b.bar = t;
    b.bar_index = LM_INDEX;
  }
}
/* The W wavefronts of a row share the highest bar that any of them knows: `top`
 * elements are not below it, wherever they are.  It is only ever raised, and
 * whoever misses a rise keeps more than it needs.  Where `top` is not small each of them
 * also leaves its m-th best element, m = top / W rounded up: no fewer than `top`
 * are not below the lowest of those, which is more than one of them finds alone
 * (4096 rows of 50257 bfloat16 with entropy: 50 alternatives 126 us, without parts 153, 20 116 and 124; for 5 it is not
 * worth its barrier). */
#define LM_WAVES (LM_LANES / 64)
#if LM_LANES > 64 && LM_TOP
static LOCAL_MEM ga_uint lm_shared_bar, lm_parts[LM_WAVES];
LM_FN void lm_reset_bar() {
  if (LID_0 < LM_WAVES) lm_shared_bar = lm_parts[LID_0] = lm_ordered(-INFINITY);
  local_barrier();
}
LM_FN void lm_heed_bar(lm_best &b) {
  lm_raise(b, __hip_atomic_load(&lm_shared_bar, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
}
LM_FN void lm_share_bar(float bar) {
  if ((LID_0 & 63) == 0) atomicMax(&lm_shared_bar, lm_ordered(bar));
}
LM_FN bool lm_by_parts(ga_int top) { return top >= 2 * LM_WAVES; }
LM_FN ga_int lm_part_of(ga_int top) { return (top + LM_WAVES - 1) / LM_WAVES; }
LM_FN void lm_leave_part(ga_uint ordered) {
  if ((LID_0 & 63) == 0) __hip_atomic_store(&lm_parts[LID_0 >> 6], ordered, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
LM_FN void lm_heed_parts(lm_best &b) {
  ga_uint t = __hip_atomic_load(&lm_parts[LID_0 & (LM_WAVES - 1)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  t = min(t, lm_xor<1>(t));
  t = min(t, lm_xor<2>(t));
  if (LM_WAVES > 4) t = min(t, lm_xor<7>(t));
  if (LM_WAVES > 8) t = min(t, lm_xor<15>(t));
  lm_raise(b, t);
}
#else
LM_FN void lm_reset_bar() {}
LM_FN void lm_heed_bar(lm_best &) {}
LM_FN void lm_share_bar(float) {}
LM_FN bool lm_by_parts(ga_int) { return false; }
LM_FN ga_int lm_part_of(ga_int top) { return top; }
LM_FN void lm_leave_part(ga_uint) {}
LM_FN void lm_heed_parts(lm_best &) {}
#endif

/* The N elements of every lane, the largest of which is `most`.  Element i of a lane has the index
 * at + (i / LM_E) * step + i % LM_E.  In a first batch the wavefronts put
 * their parts together; elsewhere, where `top` lanes or more have one that passes
 * the bar, the bar rises to the top-th largest of the lanes' largest: there are
 * that many elements that are not below it.  So a first batch, or a
 * row that rises, lets little more than `top` elements pass.  Then in rounds:
 * each lane's largest goes to wait if it passes the bar, until none does. */
template <int N> LM_FN void lm_offer(lm_best &b, float (&y)[N], float most, ga_int top, ga_uint at, ga_uint step, bool first) {
  const ga_uint lane = LID_0 & 63;
  const bool parts = lm_by_parts(top);
  if (first && parts) {
    lm_leave_part(lm_kth(lm_ordered(most), lm_part_of(top)));
    local_barrier();
    lm_heed_parts(b);
  } else {
    lm_heed_bar(b);
  }
  const ga_ulong pass = __builtin_amdgcn_ballot_w64((most > b.bar) | ((most == b.bar) & (at < b.bar_index)));
  if (pass == 0) return;
  if (__builtin_popcountll(pass) >= top && !(first && parts)) lm_raise(b, lm_kth(lm_ordered(most), top));
  do {
    int best = N - 1;
#pragma unroll
    for (int i = N - 2; i >= 0; i--) best = y[i] == most ? i : best;
    const ga_uint index = at + (ga_uint)(best / LM_E) * step + (ga_uint)(best % LM_E);
    const bool passes = (most > b.bar) | ((most == b.bar) & (index < b.bar_index));
    const ga_ulong all = __builtin_amdgcn_ballot_w64(passes);
    if (all == 0) break;
    const ga_uint count = (ga_uint)__builtin_popcountll(all);
    if (b.n + count > 64) lm_settle(b, top);
    /* those that pass go to lanes n, n + 1, ..; the others behind them, all lanes round */
    const ga_uint before = __builtin_amdgcn_mbcnt_hi((ga_uint)(all >> 32), __builtin_amdgcn_mbcnt_lo((ga_uint)all, 0));
    const int to = (int)((b.n + (passes ? before : count + lane - before)) << 2);
    const ga_ulong key = lm_key(most, index);
    const ga_uint lo = (ga_uint)__builtin_amdgcn_ds_permute(to, (int)(ga_uint)key);
    const ga_uint hi = (ga_uint)__builtin_amdgcn_ds_permute(to, (int)(ga_uint)(key >> 32));
    if (lane - b.n < count) b.waiting = (ga_ulong)hi << 32 | lo;
    b.n = (ga_uint)__builtin_amdgcn_readfirstlane((int)(b.n + count));
    best = passes ? best : N;
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = best == i ? -INFINITY : y[i];
    most = lm_max_of(y, -INFINITY);
  } while (__builtin_amdgcn_ballot_w64(most >= b.bar) != 0);
  if (parts && b.n >= 32) {
    lm_settle(b, top);
    const ga_ulong k = lm_lane(b.list, lm_part_of(top) - 1);
    if (k != 0) lm_leave_part((ga_uint)(k >> 30));
    lm_heed_parts(b);
  }
  lm_share_bar(b.bar);
}

/* The token of a row and its logit, which are fetched before the row is summed. */
struct lm_token {
  ga_long id;   /* -1: no token, -2: out of range */
  float x;
};
LM_FN LM_ID lm_token_id(const lm_logprobs &p, ga_long r) {
  return p.ids != nullptr ? *lm_at(p.ids, r * p.id_step) : 0;
}
LM_FN lm_token lm_token_of(const lm_logprobs &p, ga_long r, LM_ID id) {
  lm_token k = {-1, 0.0f};
  if (p.ids != nullptr) {
    k.id = lm_id(id, p.ignore, LM_NONE, p.v);
    k.x = lm_get(lm_at(p.logits, r * p.row)[k.id > 0 ? k.id : 0]);
  }
  return k;
}
/* log p of an element: scale * (x - m) - ls, by halves, as the difference itself may be in no float */
LM_FN float lm_logp(float x, float half_m, float scale, float ls) {
  return __builtin_fmaf(__builtin_fmaf(x, 0.5f, -half_m) * scale, 2.0f, -ls);
}
/* What is written for row r; a whole wavefront. */
LM_FN void lm_logprobs_finish(const lm_logprobs &p, ga_long r, const lm_state &a, ga_ulong list, lm_token token) {
  const ga_uint lane = LID_0 & 63;
  const float rm = a.m * p.by;
  const bool nothing = a.s == 0.0f;
  const float s = a.m == INFINITY ? NAN : a.s;
  const float m = nothing ? -INFINITY : a.m, half_m = 0.5f * m;
  const float lg = __builtin_logf(s);
  /* R(m) is off by * m by a rounding; past LM_FAR the sum is relative to m itself */
  const float off = __builtin_fabsf(rm) <= LM_FAR ? __builtin_fmaf(a.m, p.by, -rm) * 0.6931471805599453f : 0.0f;
  const float ls = nothing ? -INFINITY : lg - off;
  if (lane == 0) {
    if (p.ids != nullptr) {
      float lp = 0.0f;
      if (token.id == -2) {
        *p.err = -1;
        lp = NAN;
      } else if (token.id >= 0) {
        lp = nothing ? -INFINITY : lm_logp(token.x, half_m, p.scale, ls);
        if (ls != ls) lp = NAN;
      }
      *lm_at(p.logp, r * p.logp_step) = lp;
    }
#if LM_ENT
    if (p.entropy != nullptr)
      *lm_at(p.entropy, r * p.entropy_step) = nothing ? 0.0f : lg - 0.6931471805599453f * (a.w / s);
#endif
    if (p.stats != nullptr) {
      *lm_at(p.stats, r * p.stats_row) = m;
      *lm_at(p.stats, r * p.stats_row + p.stats_col) = ls;
    }
  }
#if LM_TOP
  const ga_ulong got = __builtin_amdgcn_ballot_w64(list != 0 && lane < p.top);
  ga_uint n = (ga_uint)__builtin_popcountll(got);
  const auto put = [&](ga_uint k, float lp, ga_uint id) {
    *lm_at(p.top_logp, r * p.topl_row + k * p.topl_col) = lp;
    const ga_long at = r * p.topi_row + k * p.topi_col;
    if (p.top_long) *lm_at((GLOBAL_MEM ga_long *)p.top_ids, at) = id;
    else *lm_at((GLOBAL_MEM ga_int *)p.top_ids, at) = (ga_int)id;
  };
  if (ls != ls) {
    if (lane < p.top) put(lane, NAN, lane);
    return;
  }
  if (lane < n) put(lane, lm_logp(lm_key_value(list), half_m, p.scale, ls), lm_key_index(list));
  /* fewer than `top` elements above -inf: the lowest indices of -inf follow.
   * They are among the first 2 * 64 elements, or the row is shorter. */
  for (ga_long base = 0; n < p.top && base < p.v; base += 64) {
    const ga_long c = base + lane;
    const bool is = c < p.v && lm_get(lm_at(p.logits, r * p.row)[c]) == -INFINITY;
    const ga_ulong hits = __builtin_amdgcn_ballot_w64(is);
    const ga_uint k = n + __builtin_amdgcn_mbcnt_hi((ga_uint)(hits >> 32), __builtin_amdgcn_mbcnt_lo((ga_uint)hits, 0));
    if (is && k < p.top) put(k, -INFINITY, (ga_uint)c);
    n += (ga_uint)__builtin_popcountll(hits);
  }
#endif
}

/* The statistics and lists of a group's wavefronts meet in the first one. */
LM_FN void lm_join_group(lm_state &a, ga_ulong &list, float by) {
  (void)list;
#if LM_WAVES > 1
  LOCAL_MEM lm_state states[LM_WAVES];
  const ga_uint wave = LID_0 >> 6, lane = LID_0 & 63;
  if (lane == 0) states[wave] = a;
#if LM_TOP
  LOCAL_MEM ga_ulong lists[LM_WAVES][64];
  lists[wave][lane] = list;
#endif
  local_barrier();
  if (wave != 0) return;
#pragma unroll
  for (int i = 1; i < LM_WAVES; i++) lm_join(a, states[i], by);
#if LM_TOP
  for (int i = 1; i < LM_WAVES; i++) lm_merge(list, lists[i][lane]);
#endif
#endif
}

template <int N> LM_FN void lm_take(lm_state &a, lm_best &best, float (&y)[N], const lm_logprobs &p, ga_uint at,
                                    ga_uint step, bool first) {
  const float most = lm_max_of(y, LM_LOWEST);
  lm_add(a, y, most, p.by);
#if LM_TOP
  /* (a lane with -inf alone offers nothing: its largest must not pass for LM_LOWEST) */
  float largest = most;
  if (__builtin_amdgcn_ballot_w64(!(most > LM_LOWEST)) != 0) largest = lm_max_of(y, -INFINITY);
  lm_offer(best, y, largest, p.top, at, step, first);
#endif
}

#if LM_SPLIT
/* The pieces of row r: a piece's statistics to a lane and its list to a
 * wavefront at a time, in fixed order. */
LM_FN void lm_join_pieces(const lm_logprobs &p, ga_long r) {
  const ga_uint wave = LID_0 >> 6, lane = LID_0 & 63;
  GLOBAL_MEM const char *from = p.partials + (ga_size)r * p.pieces * p.partial_bytes;
  lm_state a = {LM_LOWEST, 0.0f, 0.0f, 0.0f};
  ga_ulong list = 0;
  /* Every load has a long way: all of them go out before the first is used. */
  const LM_ID token_id = lm_token_id(p, r);
  const auto word = [&](ga_uint i, ga_uint place) {
    return lm_fetch((GLOBAL_MEM const ga_ulong *)(from + (ga_size)(i < p.pieces ? i : 0) * p.partial_bytes) + place);
  };
  ga_ulong ms = word(LID_0, 0), ws = word(LID_0, 1);
#if LM_TOP
  const ga_uint place = 2 + (lane < p.top ? lane : 0);
  ga_ulong k[8];     /* the lists: pieces wave, wave + LM_WAVES, .. to each wavefront */
#pragma unroll
  for (int u = 0; u < 8; u++) k[u] = word(wave + u * LM_WAVES, place);
#endif
  const lm_token token = lm_token_of(p, r, token_id);
  for (ga_uint i = LID_0; i < p.pieces; i += LM_LANES) {
    if (i != LID_0) {
      ms = word(i, 0);
      ws = word(i, 1);
    }
    const lm_state b = {__builtin_bit_cast(float, (ga_uint)ms), __builtin_bit_cast(float, (ga_uint)(ms >> 32)),
                        __builtin_bit_cast(float, (ga_uint)ws), 0.0f};
    lm_join(a, b, p.by);
  }
  lm_join_wave(a, p.by);
#if LM_TOP
  for (ga_uint i0 = wave; i0 < p.pieces; i0 += 8 * LM_WAVES) {
    if (i0 != wave) {
#pragma unroll
      for (int u = 0; u < 8; u++) k[u] = word(i0 + u * LM_WAVES, place);
    }
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (i0 + u * LM_WAVES < p.pieces) lm_merge(list, lane < p.top ? k[u] : 0);
  }
#endif
  local_barrier();   /* (the group's LDS is free again) */
  lm_join_group(a, list, p.by);
  if (wave == 0) lm_logprobs_finish(p, r, a, list, token);
}
#endif

#define LM_U (16 / LM_E)   /* chunks of a lane at a time: 16 elements */

/* One pass over the row with the running maximum and sums; what an element costs is a
 * multiply-add, an exponential and an addition, one more multiply-add with the entropy, and half a
 * maximum.  4096 rows of 50257 bfloat16 with entropy take 67 to 69 us (412 MB, 6.0 TB/s) where the vector
 * instructions alone take about 52; 65536 rows of 1000 floats with 5 alternatives 58 to 63 us
 * (262 MB, 4.3 TB/s): a wavefront sees its row in one batch, and the alternatives' networks and rounds
 * are half of its instructions.
 *
 * LM_LANES lanes share a row, or one of its pieces (LM_SPLIT): a loop over
 * the row's aligned 16-byte chunks, LM_U per lane at a time, the next ones
 * loading while the present ones are summed.  The elements before the first
 * and after the last whole chunk go one to a lane. */
#if LM_TOP && LM_ENT && LM_LANES == 256   /* (96 registers, which are enough: five wavefronts on a SIMD, not four) */
#define LM_OCC __attribute__((amdgpu_waves_per_eu(5)))
#else
#define LM_OCC
#endif
KERNEL void __launch_bounds__(LM_LANES < 256 ? 256 : LM_LANES) LM_OCC lm_logprobs_rows(const lm_logprobs p) {
#if LM_LANES < 256
  const ga_long r = (ga_long)GID_0 * (256 / LM_LANES) + __builtin_amdgcn_readfirstlane((int)(LID_0 / LM_LANES));
  if (r >= p.t) return;
  const ga_uint lane = LID_0 % LM_LANES;
#else
  const ga_uint lane = LID_0;
#if LM_SPLIT
  const ga_long r = GID_0 / p.pieces;
#else
  const ga_long r = GID_0;
#endif
#endif
#if LM_SPLIT
  const ga_uint piece = GID_0 % p.pieces;
#else
  const ga_uint piece = 0;
#endif
  GLOBAL_MEM const LM_X *x = lm_at(p.logits, r * p.row);
  const ga_uint v = (ga_uint)p.v;
  ga_uint head = (ga_uint)(-(ga_size)x & 15) / (ga_uint)sizeof(LM_X);
  if (head > v) head = v;
  const ga_uint chunks = (v - head) / LM_E;
  const ga_uint tail0 = head + chunks * LM_E;
  GLOBAL_MEM const lm_u4 *q = (GLOBAL_MEM const lm_u4 *)(x + head);
#if LM_SPLIT
  const ga_uint from = piece * p.piece_chunks;
  const ga_uint to = from + p.piece_chunks < chunks ? from + p.piece_chunks : chunks;
#else
  const ga_uint from = 0, to = chunks;
#endif
  const ga_uint minus_inf = lm_minus_inf(LM_X());
  lm_state a = {LM_LOWEST, 0.0f, 0.0f, 0.0f};
  lm_best best = {0, 0, 0, 0, -INFINITY};
#if !LM_SPLIT
  const LM_ID token_id = lm_token_id(p, r);
#endif
  lm_u4 raw[LM_U];
  const auto fetch = [&](ga_uint base) {   /* unconditional loads: all of them in flight */
    if (base + LM_U * LM_LANES <= to) {
#pragma unroll
      for (int u = 0; u < LM_U; u++) raw[u] = __builtin_nontemporal_load(q + (base + u * LM_LANES + lane));
    } else {
#pragma unroll
      for (int u = 0; u < LM_U; u++) {
        const ga_uint c = base + u * LM_LANES + lane;
        raw[u] = __builtin_nontemporal_load(q + (c < to ? c : to - 1));
      }
#pragma unroll
      for (int u = 0; u < LM_U; u++) {
        const bool in = base + u * LM_LANES + lane < to;
#pragma unroll
        for (int i = 0; i < 4; i++) raw[u][i] = in ? raw[u][i] : minus_inf;
      }
    }
  };
  if (from < to) fetch(from);
  lm_reset_bar();
#if !LM_SPLIT
  const lm_token token = lm_token_of(p, r, token_id);
#endif
  for (ga_uint base = from; base < to; base += LM_U * LM_LANES) {
    const ga_uint at = head + (base + lane) * LM_E;
    if (base + (lane & ~63u) + LM_LANES < to) {
      float y[LM_U * LM_E];
#pragma unroll
      for (int u = 0; u < LM_U; u++) lm_unpack(raw[u], y + u * LM_E, LM_X());
      if (base + LM_U * LM_LANES < to) fetch(base + LM_U * LM_LANES);
      lm_take(a, best, y, p, at, LM_LANES * LM_E, base == from);
    } else {          /* the last ones: no more than one chunk for any lane of this wavefront */
      float y[LM_E];
      lm_unpack(raw[0], y, LM_X());
      lm_take(a, best, y, p, at, LM_LANES * LM_E, base == from);
    }
  }
  /* (last, so that the bar of the alternatives comes from a full batch) */
  if (piece == 0 && lane < 64 && v != chunks * LM_E) {
    float y[1] = {-INFINITY};
    ga_uint c = lane < head ? lane : tail0 + (lane - head);
    if (c < v) y[0] = lm_get(x[c]);
    lm_take(a, best, y, p, c, 0, false);
  }
  lm_join_wave(a, p.by);
  lm_settle(best, p.top);
  ga_ulong list = best.list;
  lm_join_group(a, list, p.by);
#if LM_SPLIT
  if (LID_0 < 64) {
    GLOBAL_MEM char *mine = p.partials + (ga_size)GID_0 * p.partial_bytes;
    GLOBAL_MEM ga_ulong *words = (GLOBAL_MEM ga_ulong *)mine;
    if (lane == 0) {
      lm_publish(words, (ga_ulong)__builtin_bit_cast(ga_uint, a.s) << 32 | __builtin_bit_cast(ga_uint, a.m));
      lm_publish(words + 1, (ga_ulong)__builtin_bit_cast(ga_uint, a.w));
    }
#if LM_TOP
    if (lane < p.top) lm_publish(words + 2 + lane, list);
#endif
  }
  LOCAL_MEM ga_uint last;
  if (LID_0 < 64) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   /* (of every lane of the wavefront) */
    if (lane == 0) last = lm_count_in(p.counters + r, p.pieces);
  }
  local_barrier();
  if (last) lm_join_pieces(p, r);
#else
  if (LID_0 < 64 || LM_WAVES == 1) lm_logprobs_finish(p, r, a, list, token);
#endif
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
  float scale, by;               /* by = scale * log2(e) */
  ga_uint segments;
};
#define LM_U (32 / LM_E)   /* chunks of a lane: 32 elements */

/* A wavefront takes 64 * LM_U chunks of a row, on the result's 16-byte
 * boundaries; what a row needs is a handful of scalars.  With
 *   a = log2 p = (by * x - R) - rest,  R = by * m rounded,  rest = (by * m - R) + log2 of the sum
 * an element is p * (A + B a), A = -scale (dlogp + dentropy * entropy), B = -scale * dentropy * ln 2, and the token's own has
 * scale * dlogp besides.  One read and one write of every element: bound by memory,
 * 4096 rows of 50257 bfloat16 149 us (824 MB, 5.5 TB/s; rows on 16-byte boundaries the same).
 * By the elements of a lane, 16, 32, 64, 128: 149, 149, 155, 165 us; 20000 rows of 1000 floats 32, 31, 31, 65. */
KERNEL void __launch_bounds__(256) lm_logprobs_grad_rows(const lm_logprobs_grad p) {
  const ga_uint unit = (ga_uint)__builtin_amdgcn_readfirstlane((int)(GID_0 * 4 + (LID_0 >> 6)));
  const ga_long r = unit / p.segments;
  if (r >= p.t) return;
  const ga_uint segment = unit % p.segments, lane = LID_0 & 63;
  GLOBAL_MEM const LM_X *x = lm_at(p.logits, r * p.row);
  GLOBAL_MEM LM_X *o = lm_at(p.out, r * p.out_row);
  const ga_int v = (ga_int)p.v;
  /* chunk c has the elements first + c * LM_E .. of the row, those that it has */
  const ga_int first = -(ga_int)(((ga_size)o & 15) / sizeof(LM_X));
  const ga_int at = first + (ga_int)((segment * 64 * LM_U + lane) * LM_E);
  /* Unconditional loads, all of them in flight: at the row's ends the first or
   * last LM_E elements, of which the lane writes those of its chunk. */
  float y[LM_U][LM_E];
  if (v >= LM_E) {
#pragma unroll
    for (int u = 0; u < LM_U; u++) {
      const ga_int c = at + u * 64 * LM_E, from = c < 0 ? 0 : c > v - LM_E ? v - LM_E : c;
      const lm_u4 q = __builtin_nontemporal_load((GLOBAL_MEM const lm_u4a *)(x + from));
      lm_unpack(q, y[u], LM_X());
    }
  } else {
#pragma unroll
    for (int u = 0; u < LM_U; u++)
#pragma unroll
      for (int e = 0; e < LM_E; e++) y[u][e] = e < v ? (float)lm_get(x[e]) : 0.0f;
  }
  const float m = *lm_at(p.stats, r * p.stats_row), ls = *lm_at(p.stats, r * p.stats_row + p.stats_col);
  float g = 0.0f, gh = 0.0f, h = 0.0f;
  ga_long id = -1;
  if (p.ids != nullptr) {
    id = lm_id(*lm_at(p.ids, r * p.id_step), p.ignore, LM_NONE, p.v);
    if (id == -2 && segment == 0 && lane == 0) *p.err = -1;
    if (id >= 0) g = *lm_at(p.dlogp, r * p.dlogp_step);
  }
#if LM_ENT
  gh = *lm_at(p.dentropy, r * p.dentropy_step);
  h = *lm_at(p.entropy, r * p.entropy_step);
#endif
  const float big = p.by * m;
  const bool nothing = ls == -INFINITY;
  const bool far = !(__builtin_fabsf(big) <= LM_FAR);   /* R is no part of the exponent then, as in the statistics */
  const float rest = (far ? 0.0f : __builtin_fmaf(p.by, m, -big)) + ls * 1.4426950408889634f;
  /* a scale that would take A out of range, and 0 * A to NaN, is multiplied in at the end */
  const bool steep = p.scale > 0x1p64f;
  const float scale = steep ? p.scale * 0x1p-64f : p.scale;
  const float a = -scale * (g + gh * h) + (ls - ls), b = -scale * gh * 0.6931471805599453f;   /* (NaN where ls is) */
  const float own = scale * g;
#pragma unroll
  for (int u = 0; u < LM_U; u++) {
    const ga_int c = at + u * 64 * LM_E;
    const ga_int from = v < LM_E || c < 0 ? 0 : c > v - LM_E ? v - LM_E : c;
    if (c >= v) break;
    float d[LM_E];
    if (nothing) {
#pragma unroll
      for (int e = 0; e < LM_E; e++) d[e] = 0.0f;
    } else {
#pragma unroll
      for (int e = 0; e < LM_E; e++) {
        float l = __builtin_fmaf(y[u][e], p.by, -big) - rest;
        if (far) l = (y[u][e] - m) * p.by - rest;
        const float q = __builtin_amdgcn_exp2f(l);
#if LM_ENT
        d[e] = q * __builtin_fmaf(b, __builtin_fmaxf(l, -300.0f), a);
#else
        d[e] = q * a;
#endif
      }
      if (id >= from && id < from + LM_E) {
#pragma unroll
        for (int e = 0; e < LM_E; e++) d[e] += from + e == id ? own : 0.0f;
      }
      if (steep) {
#pragma unroll
        for (int e = 0; e < LM_E; e++) d[e] *= 0x1p64f;
      }
    }
    if (from == c && v >= LM_E) {
      lm_store(o + c, d);
    } else {
#pragma unroll
      for (int e = 0; e < LM_E; e++)
        if (from + e >= c && from + e < c + LM_E && from + e < v) lm_put(o + from + e, d[e]);
    }
  }
}
#endif

#if LM_KIND == LM_K_NORM || LM_KIND == LM_K_CLIP
/* The arrays of a launch, cut in pieces of `piece` 16-byte chunks that are
 * numbered through; `first` is the number of an array's first piece.  They come
 * with the arguments, up to LM_TENSORS of them, or lie in a table in device
 * memory (LM_TENSORS 0).  A piece finds its array with one load a lane and a ballot, for each
 * factor of 64 in their number. */
struct lm_tensor {
  GLOBAL_MEM const void *in;
  GLOBAL_MEM void *out;
  ga_long count;
  ga_uint first, type;           /* type: 0 float, 1 half, 2 bfloat16, 3 double */
};
struct lm_tensors {
  GLOBAL_MEM double *partials;   /* sums of squares, one per group; `ends` later, of the large and the small ones */
  GLOBAL_MEM double *result;     /* the factor, the norm */
  GLOBAL_MEM void *norm;
  GLOBAL_MEM ga_uint *counter;   /* a zero that the last table's groups count on; NULL for the others */
  double max_norm;
  ga_uint partial0, npartials;
  ga_uint n, pieces, piece;
  ga_int norm_double;
  ga_uint ends, pad;             /* (of LM_ENDS) */
#if LM_TENSORS
  lm_tensor tensors[LM_TENSORS];
#else
  GLOBAL_MEM const lm_tensor *tensors;
#endif
};
LM_FN ga_uint lm_find(const lm_tensors &p, ga_uint piece) {
  ga_uint from = 0, n = p.n;
  while (n > 1) {
    const ga_uint step = (n + 63) / 64, i = (LID_0 & 63) * step;
    const bool begun = i < n && p.tensors[from + (i < n ? i : 0)].first <= piece;
    const ga_uint at = ((ga_uint)__builtin_popcountll(__builtin_amdgcn_ballot_w64(begun)) - 1) * step;
    from += at;
    n = n - at < step ? n - at : step;
  }
  return (ga_uint)__builtin_amdgcn_readfirstlane((int)from);
}
#define LM_GROUP 256
#define LM_BY_TYPE(type, F)       \
  switch (type) {                 \
    case 0: F(ga_float); break;   \
    case 1: F(ga_half); break;    \
    case 2: F(ga_bfloat16); break; \
    LM_DOUBLES(F)                 \
  }
#if LM_KIND == LM_K_CLIP || LM_ENDS
#define LM_DOUBLES(F) default: F(ga_double); break;
#else
#define LM_DOUBLES(F)
#endif
LM_FN double lm_lane_xor(double v, int mask) {
  const ga_ulong b = __builtin_bit_cast(ga_ulong, v);
  const int from = (int)(((LID_0 & 63) ^ mask) << 2);
  const ga_uint lo = (ga_uint)__builtin_amdgcn_ds_bpermute(from, (int)(ga_uint)b);
  const ga_uint hi = (ga_uint)__builtin_amdgcn_ds_bpermute(from, (int)(ga_uint)(b >> 32));
  return __builtin_bit_cast(double, (ga_ulong)hi << 32 | lo);
}
LM_FN double lm_wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += lm_lane_xor(v, d);
  return v;
}
LM_FN void lm_unpack(const lm_u4 &q, double *y, ga_double) {
  typedef double d2 __attribute__((ext_vector_type(2)));
  const d2 d = __builtin_bit_cast(d2, q);
  y[0] = d[0];
  y[1] = d[1];
}
template <class T> struct lm_wide { typedef float type; };
template <> struct lm_wide<ga_double> { typedef double type; };
#endif

#if LM_KIND == LM_K_NORM
#define LM_U 8   /* chunks in flight per lane */

/* Sums of squares in 64 bits: a multiply-add of doubles costs what one of floats does, and neither the
 * largest nor the smallest float's square leaves their range.  A double's may.  Where there are doubles
 * (LM_ENDS) those past 2^486 and those below 2^-511 are summed on their own, multiplied by 2^-600 or 2^600, so that no sum of
 * up to 2^50 squares overflows and none that counts is lost (three sums, as J. L. Blue has them, 1978).  Hardly any
 * array has such numbers: a look at the upper words of a batch finds them, and what has none
 * leaves and fetches one sum, whose sign says so (75 million doubles 105.6 us, unscaled 103.9; 3000 4.8 and 4.2). */
struct lm_sums {
  double s;
#if LM_ENDS
  double large, small;
#endif
};
template <int N> LM_FN void lm_add_squares(lm_sums &, double (&s)[4], const float (&y)[N]) {
#pragma unroll
  for (int e = 0; e < N; e++) s[e & 3] = __builtin_fma((double)y[e], (double)y[e], s[e & 3]);
}
#if LM_ENDS
#define LM_LARGE 0x1p486
#define LM_SMALL 0x1p-511
#define LM_DOWN 0x1p-600
#define LM_UP 0x1p600
template <int N> LM_FN void lm_add_squares(lm_sums &t, double (&s)[4], const double (&y)[N]) {
  bool far = false;
#pragma unroll
  for (int e = 0; e < N; e++)   /* the upper words of 2^-511 and 2^486 */
    far |= ((ga_uint)(__builtin_bit_cast(ga_ulong, y[e]) >> 32) & 0x7fffffffu) - 0x20000000u >= 0x5e500000u - 0x20000000u;
  if (__builtin_amdgcn_ballot_w64(far) == 0) {
#pragma unroll
    for (int e = 0; e < N; e++) s[e & 3] = __builtin_fma(y[e], y[e], s[e & 3]);
    return;
  }
#pragma unroll
  for (int e = 0; e < N; e++) {
    const double a = __builtin_fabs(y[e]), l = a > LM_LARGE ? y[e] * LM_DOWN : 0.0, m = a < LM_SMALL ? y[e] * LM_UP : 0.0;
    const double c = a > LM_LARGE || a < LM_SMALL ? 0.0 : y[e];
    t.large = __builtin_fma(l, l, t.large);
    t.small = __builtin_fma(m, m, t.small);
    s[e & 3] = __builtin_fma(c, c, s[e & 3]);
  }
}
LM_FN bool lm_ends(const lm_sums &t) { return t.large != 0.0 || t.small != 0.0; }
LM_FN double lm_marked(double s, bool ends) { return __builtin_copysign(s, ends ? -1.0 : 1.0); }
LM_FN bool lm_is_marked(double s) { return (__builtin_bit_cast(ga_ulong, s) >> 63) != 0; }
#endif
/* the sums over a group */
LM_FN lm_sums lm_group_sum(lm_sums t) {
  LOCAL_MEM double part[LM_GROUP / 64];
  t.s = lm_wave_sum(t.s);
#if LM_ENDS
  LOCAL_MEM double large[LM_GROUP / 64], small[LM_GROUP / 64];
  const bool ends = __builtin_amdgcn_ballot_w64(lm_ends(t)) != 0;
  t.s = lm_marked(t.s, ends);
  if (ends) {
    t.large = lm_wave_sum(t.large);
    t.small = lm_wave_sum(t.small);
    if ((LID_0 & 63) == 0) large[LID_0 >> 6] = t.large, small[LID_0 >> 6] = t.small;
  }
#endif
  if ((LID_0 & 63) == 0) part[LID_0 >> 6] = t.s;
  local_barrier();
#if LM_ENDS
  t.s = t.large = t.small = 0.0;
#pragma unroll
  for (int w = 0; w < LM_GROUP / 64; w++) {
    t.s += __builtin_fabs(part[w]);
    if (lm_is_marked(part[w])) t.large += large[w], t.small += small[w];
  }
#else
  t.s = part[0];
#pragma unroll
  for (int w = 1; w < LM_GROUP / 64; w++) t.s += part[w];
#endif
  return t;
}
/* The squares of n elements of type T. */
template <class T> LM_FN void lm_squares(lm_sums &t, GLOBAL_MEM const T *x, ga_long n) {
  constexpr int E = 16 / (int)sizeof(T);
  typedef typename lm_wide<T>::type wide;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  ga_long head = (ga_long)((-(ga_size)x & 15) / sizeof(T));
  if (head > n) head = n;
  const ga_uint whole = (ga_uint)((n - head) / E);
  const ga_long tail = head + (ga_long)whole * E;
  GLOBAL_MEM const lm_u4 *q = (GLOBAL_MEM const lm_u4 *)(x + head);
  const ga_long k = LID_0 < head ? (ga_long)LID_0 : tail + (LID_0 - head);
  if (k < n) {
    const wide y[1] = {lm_get(x[k])};
    lm_add_squares(t, s, y);
  }
  lm_u4 raw[LM_U];
  ga_uint c0 = 0;
  for (; c0 + LM_GROUP * LM_U <= whole; c0 += LM_GROUP * LM_U) {
    wide y[LM_U * E];
#pragma unroll
    for (int u = 0; u < LM_U; u++) raw[u] = q[c0 + u * LM_GROUP + LID_0];
#pragma unroll
    for (int u = 0; u < LM_U; u++) lm_unpack(raw[u], y + u * E, T());
    lm_add_squares(t, s, y);
  }
  if (c0 < whole) {     /* (unconditional loads: all of them in flight) */
#pragma unroll
    for (int u = 0; u < LM_U; u++) {
      const ga_uint c = c0 + u * LM_GROUP + LID_0;
      raw[u] = q[c < whole ? c : whole - 1];
    }
#pragma unroll
    for (int u = 0; u < LM_U; u++) {
      wide y[E];
      lm_unpack(raw[u], y, T());
      if (c0 + u * LM_GROUP + LID_0 < whole) lm_add_squares(t, s, y);
    }
  }
  t.s += (s[0] + s[1]) + (s[2] + s[3]);
}
/* The norm and the factor from all partial sums, by one group. */
LM_FN void lm_norm_of_partials(const lm_tensors &p) {
  lm_sums t = {};
  const auto part = [&](ga_uint k) { return __builtin_bit_cast(double, lm_fetch((GLOBAL_MEM const ga_ulong *)p.partials + k)); };
  for (ga_uint k = LID_0; k < p.npartials; k += LM_GROUP) {
#if LM_ENDS
    const double s = part(k);
    t.s += __builtin_fabs(s);
    if (lm_is_marked(s)) t.large += part(p.ends + k), t.small += part(2 * p.ends + k);
#else
    t.s += part(k);
#endif
  }
  local_barrier();   /* (the LDS of an earlier sum is free again) */
  t = lm_group_sum(t);
  double norm = __builtin_sqrt(t.s);
#if LM_ENDS
  if (t.large != 0.0) norm = __builtin_sqrt(t.s * LM_DOWN * LM_DOWN + t.large) * LM_UP;
  else if (t.s == 0.0) norm = __builtin_sqrt(t.small) * LM_DOWN;
  else if (t.small != 0.0) norm = __builtin_sqrt(t.s + t.small * LM_DOWN * LM_DOWN);
#endif
  if (LID_0 == 0) {
    p.result[0] = norm > p.max_norm && norm < (double)INFINITY ? p.max_norm / norm : 1.0;
    p.result[1] = norm;
    if (p.norm != nullptr) {
      if (p.norm_double) *(GLOBAL_MEM double *)p.norm = norm;
      else *(GLOBAL_MEM float *)p.norm = (float)norm;
    }
  }
}
/* A group adds a range of pieces: what of it lies in one array in one go.  600 MB
 * of bfloat16 in 148 arrays take 107 us (5.6 TB/s; the vector units are busy a quarter of that); 256 to 2048
 * groups, ranges or interleaved blocks of 1 to 16 pieces, streaming loads or none: no faster. */
KERNEL void __launch_bounds__(LM_GROUP) lm_norm_pieces(const lm_tensors p) {
  lm_sums sums = {};
  const ga_uint share = (p.pieces + GDIM_0 - 1) / GDIM_0;
  ga_uint piece = GID_0 * share;
  const ga_uint end = p.pieces - piece < share ? p.pieces : piece + share;
  if (piece < p.pieces) {
    for (ga_uint i = lm_find(p, piece); piece < end; i++) {
      const lm_tensor t = p.tensors[i];
      const ga_uint next = i + 1 < p.n ? p.tensors[i + 1].first : p.pieces;
      const ga_uint stop = next < end ? next : end;
#define LM_SQUARES(T)                                                             \
  {                                                                               \
    const ga_long per = (ga_long)p.piece * (16 / (ga_long)sizeof(T));             \
    const ga_long from = (ga_long)(piece - t.first) * per, left = t.count - from; \
    const ga_long n = (ga_long)(stop - piece) * per;                              \
    lm_squares(sums, (GLOBAL_MEM const T *)t.in + from, left < n ? left : n);     \
  }
      LM_BY_TYPE(t.type, LM_SQUARES)
      piece = stop;
    }
  }
  sums = lm_group_sum(sums);
  LOCAL_MEM ga_uint last;
  if (LID_0 == 0) {
    GLOBAL_MEM ga_ulong *mine = (GLOBAL_MEM ga_ulong *)p.partials + p.partial0 + GID_0;
#if LM_ENDS
    const bool ends = lm_ends(sums);
    if (ends) {
      lm_publish(mine + p.ends, __builtin_bit_cast(ga_ulong, sums.large));
      lm_publish(mine + 2 * p.ends, __builtin_bit_cast(ga_ulong, sums.small));
    }
    sums.s = lm_marked(sums.s, ends);
#endif
    lm_publish(mine, __builtin_bit_cast(ga_ulong, sums.s));
    last = p.counter != nullptr && lm_count_in(p.counter, GDIM_0);
  }
  local_barrier();
  if (last) lm_norm_of_partials(p);
}
#endif

#if LM_KIND == LM_K_CLIP
#define LM_U 4

LM_FN void lm_scaled(const lm_u4 &q, lm_u4a &r, double by, ga_double) {
  typedef double d2 __attribute__((ext_vector_type(2)));
  d2 d = __builtin_bit_cast(d2, q);
  d[0] *= by;
  d[1] *= by;
  r = __builtin_bit_cast(lm_u4a, d);
}
template <class T> LM_FN void lm_scaled(const lm_u4 &q, lm_u4a &r, double by, T) {
  constexpr int E = 16 / (int)sizeof(T);
  float y[E];
  lm_unpack(q, y, T());
#pragma unroll
  for (int e = 0; e < E; e++) y[e] *= (float)by;
  ga_uint w[4];
  lm_pack(y, w, 4, T());
  r = lm_u4a{w[0], w[1], w[2], w[3]};
}
template <class T> LM_FN void lm_scale(GLOBAL_MEM const T *x, GLOBAL_MEM T *o, ga_long n, double by) {
  constexpr int E = 16 / (int)sizeof(T);
  ga_long head = (ga_long)((-(ga_size)o & 15) / sizeof(T));   /* chunks on the result's 16-byte boundaries */
  if (head > n) head = n;
  const ga_uint whole = (ga_uint)((n - head) / E);
  const ga_long tail = head + (ga_long)whole * E;
  const ga_long k = LID_0 < head ? (ga_long)LID_0 : tail + (LID_0 - head);
  if (k < n) lm_put(o + k, (typename lm_wide<T>::type)by * lm_get(x[k]));
  for (ga_uint c0 = 0; c0 < whole; c0 += LM_GROUP * LM_U) {
    lm_u4 raw[LM_U];     /* (unconditional loads: all of them in flight) */
#pragma unroll
    for (int u = 0; u < LM_U; u++) {
      const ga_uint c = c0 + u * LM_GROUP + LID_0;
      raw[u] = __builtin_nontemporal_load((GLOBAL_MEM const lm_u4a *)(x + head + (ga_long)(c < whole ? c : whole - 1) * E));
    }
#pragma unroll
    for (int u = 0; u < LM_U; u++) {
      const ga_uint c = c0 + u * LM_GROUP + LID_0;
      lm_u4a r;
      lm_scaled(raw[u], r, by, T());
      if (c < whole) __builtin_nontemporal_store(r, (GLOBAL_MEM lm_u4a *)(o + head + (ga_long)c * E));
    }
  }
}
/* Where the factor is below the smallest normal number of the type it is multiplied in, it has few bits left, or none:
 * x / norm, 1 at most, times max_norm has all of them.  (A max_norm of 0 is a factor like others.) */
template <class T> LM_FN bool lm_far_below(double by, double max_norm) {
  return by < (sizeof(T) == 8 ? 0x1p-1022 : 0x1p-126) && max_norm != 0.0;
}
template <class T> LM_FN void lm_scale_far(GLOBAL_MEM const T *x, GLOBAL_MEM T *o, ga_long n, double norm, double max_norm) {
  for (ga_long k = LID_0; k < n; k += LM_GROUP)
    lm_put(o + k, (typename lm_wide<T>::type)((double)lm_get(x[k]) / norm * max_norm));
}
/* A group for each piece.  600 MB of bfloat16: 189 us, 6.4 TB/s of reads and writes.  Where
 * nothing is clipped in place nothing is read. */
KERNEL void __launch_bounds__(LM_GROUP) lm_clip_pieces(const lm_tensors p) {
  const ga_uint piece = GID_0;
  const lm_tensor t = p.tensors[lm_find(p, piece)];
  const double by = p.result[0];
  if (by == 1.0 && t.in == t.out) return;
#define LM_SCALE(T)                                                          \
  {                                                                          \
    const ga_long per = (ga_long)p.piece * (16 / (ga_long)sizeof(T));        \
    const ga_long from = (ga_long)(piece - t.first) * per, left = t.count - from; \
    GLOBAL_MEM const T *x = (GLOBAL_MEM const T *)t.in + from;               \
    GLOBAL_MEM T *o = (GLOBAL_MEM T *)t.out + from;                          \
    if (lm_far_below<T>(by, p.max_norm)) lm_scale_far(x, o, left < per ? left : per, p.result[1], p.max_norm); \
    else lm_scale(x, o, left < per ? left : per, by);                        \
  }
  LM_BY_TYPE(t.type, LM_SCALE)
}
#endif
