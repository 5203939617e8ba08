// Operators of language models: embedding rows and their gradient, log
// probabilities of tokens and their gradient, the global norm of many arrays
// and clipping by it.  The rules are those of gpuarray/language.h; the kernels
// are in language_kernels.h and are compiled per operator and set of types,
// kept for the life of the context like those of GpuArray_take1.
#include "private.hpp"

#include <algorithm>
#include <cmath>
#include <memory>
#include <string>
#include <unordered_map>
#include <vector>

namespace {

// ---- kernels of a context ------------------------------------------------------

enum lm_kind { LM_EMBED, LM_EMBED_GRAD, LM_LOGPROBS, LM_LOGPROBS_GRAD, LM_NORM, LM_CLIP, LM_SORT };

// What a kernel text is specialised on; packed into the key it is kept under.
struct lm_variant {
  unsigned kind, x, o, id;   // operator; typecodes of operand, result, ids
  unsigned extra;            // the operator's own
  unsigned long long key() const {
    return (unsigned long long)kind | (unsigned long long)x << 8 | (unsigned long long)o << 20 |
           (unsigned long long)id << 32 | (unsigned long long)extra << 44;
  }
  explicit lm_variant(unsigned long long k)
      : kind(k & 0xff), x(k >> 8 & 0xfff), o(k >> 20 & 0xfff), id(k >> 32 & 0xfff), extra((unsigned)(k >> 44)) {}
  lm_variant(unsigned kind_, int x_, int o_, int id_, unsigned extra_)
      : kind(kind_), x((unsigned)x_), o((unsigned)o_), id((unsigned)id_), extra(extra_) {}
};

const unsigned LM_TENSORS = 112;   // arrays per launch of the norm and clip kernels

// Arguments of the kernels, as language_kernels.h declares them.
struct embed_args {
  void *out;
  const void *table, *ids;
  void *err;
  int64_t out_row, table_row, id_step;
  int64_t n, v, d, ignore;
  float scale;
  uint32_t lanes_log2, segments;
};
struct sorting_args {
  const void *ids, *key_in, *order_in;
  void *key, *order, *counts, *err;
  int64_t id_step, ignore, v;
  uint32_t n, groups, shift, bits, passes, direct;
  void *fill;
  int64_t fill_rows, fill_row, fill_bytes, fill_unit0, fill_unit1;
};
struct embed_grad_args {
  void *grad;
  const void *dout, *key, *order;
  void *partials;
  const void *ids;
  void *err;
  int64_t id_step, ignore;
  int64_t grad_row, dout_row, v, d;
  float scale;
  int32_t accumulate;
  uint32_t n, chunk, chunks, tiles, rows, lanes_log2, dense, part_tiles;
};
struct logprobs_args {
  const void *logits, *ids;
  void *logp, *entropy, *stats, *top_logp, *top_ids;
  void *err;
  void *partials;
  int64_t row, id_step, logp_step, entropy_step, stats_row, stats_col;
  int64_t topl_row, topl_col, topi_row, topi_col;
  int64_t t, v, ignore;
  float scale, by;
  int32_t top, top_long;
  uint32_t pieces, piece_chunks, partial_bytes, pad;
  void *counters;
};
// What the variant of the log probability kernels is specialised on: the lanes
// of a row, the entropy, the alternatives, rows in pieces.
inline unsigned logprobs_extra(unsigned lanes, bool entropy, bool top, bool split) {
  return lanes / 64 | (entropy ? 32u : 0) | (top ? 64u : 0) | (split ? 128u : 0);
}
struct logprobs_grad_args {
  void *out;
  const void *logits, *ids, *stats, *dlogp, *entropy, *dentropy;
  void *err;
  int64_t out_row, row, id_step, stats_row, stats_col, dlogp_step, entropy_step, dentropy_step;
  int64_t t, v, ignore;
  float scale, by;
  uint32_t segments;
};
struct tensor_arg {
  const void *in;
  void *out;
  int64_t count;
  uint32_t first, type;
};
struct norm_args {      // followed by the arrays themselves, or the address of their table
  void *partials, *result, *norm, *counter;
  double max_norm;
  uint32_t partial0, npartials, n, pieces, piece;
  int32_t norm_double;
  uint32_t ends, pad;
};
struct tensors_args {
  norm_args a;
  tensor_arg tensors[LM_TENSORS];
};
struct table_args {
  norm_args a;
  const void *tensors;
};

std::string lm_source(const lm_variant &v) {
  std::string s = "#define LM_KIND " + std::to_string(v.kind) + "\n";
  auto name = [&](const char *what, unsigned tc) {
    const char *c = gpuarray_get_type((int)tc)->cluda_name;
    s += std::string("#define ") + what + " " + (c ? c : "ga_float") + "\n";
  };
  name("LM_X", v.x);
  name("LM_O", v.o);
  name("LM_ID", v.id);
  if (v.kind == LM_EMBED_GRAD) s += std::string("#define LM_NARROW ") + (v.extra ? "1\n" : "0\n");
  if (v.kind == LM_SORT) s += "#define LM_R " + std::to_string(v.extra ? v.extra : 4) + "\n";
  if (v.kind == LM_NORM || v.kind == LM_CLIP) s += "#define LM_TENSORS " + std::to_string(v.extra & 1 ? 0 : LM_TENSORS) + "\n";
  if (v.kind == LM_NORM) s += std::string("#define LM_ENDS ") + (v.extra & 2 ? "1\n" : "0\n");
  if (v.kind == LM_LOGPROBS_GRAD) s += std::string("#define LM_ENT ") + (v.extra ? "1\n" : "0\n");
  if (v.kind == LM_LOGPROBS) {
    s += "#define LM_LANES " + std::to_string((v.extra & 31 ? v.extra & 31 : 1) * 64) + "\n";
    s += std::string("#define LM_ENT ") + (v.extra & 32 ? "1" : "0") + "\n#define LM_TOP " + (v.extra & 64 ? "1" : "0") +
         "\n#define LM_SPLIT " + (v.extra & 128 ? "1" : "0") + "\n";
  }
  return s + ga_language_kernels_src;
}

typedef std::unordered_map<std::string, GpuKernel> lm_cache;

// The kernel `name` of a variant, from the context's cache or built.  Building
// loads a code object, which a stream that records a graph does not allow.
int lm_kernel(gpucontext *ctx, const lm_variant &v, const char *name, size_t args_size, GpuKernel **out) {
  void **slot = ga_hip_language_cache_slot(ctx);
  if (*slot == nullptr) *slot = new lm_cache();
  lm_cache &cache = *(lm_cache *)*slot;
  const unsigned long long k = v.key();
  std::string key((const char *)&k, sizeof(k));
  key += name;
  auto it = cache.find(key);
  if (it != cache.end()) {
    *out = &it->second;
    return GA_NO_ERROR;
  }
  if (ga_hip_capturing(ctx))
    return ga_err_fmt(ctx->err, GA_UNSUPPORTED_ERROR,
                      "%s is not built yet and the stream records a graph: call once before recording", name);
  const std::string s = lm_source(v);
  const char *strs[1] = {s.c_str()};
  size_t lens[1] = {s.size()};
  const int types[1] = {ga_plan_typecode(args_size)};
  GpuKernel nk = {nullptr, nullptr};
  const int err = GpuKernel_init(&nk, ctx, 1, strs, lens, name, 1, types, 0, nullptr);
  if (err != GA_NO_ERROR) return err;
  *out = &cache.emplace(key, nk).first->second;
  return GA_NO_ERROR;
}

int lm_launch(GpuKernel *k, size_t groups, size_t lanes, void *args) {
  void *argv[1] = {args};
  return GpuKernel_call(k, 1, &groups, &lanes, 0, argv);
}

// `bytes` of the context's scratch.
int lm_scratch(gpucontext *ctx, size_t bytes, char **out) {
  if (bytes > ga_hip_scratch_size(ctx) && ga_hip_capturing(ctx))
    return ga_err_set(ctx->err, GA_UNSUPPORTED_ERROR,
                      "The scratch has to grow and the stream records a graph: call once before recording");
  gpudata *b = ga_hip_scratch(ctx, bytes);
  if (b == nullptr) return ctx->err->code;
  *out = (char *)b->devptr;
  return GA_NO_ERROR;
}

// The context's counters, zeros that the groups of a launch count on and that the last one zeroes.
int lm_counters(gpucontext *ctx, void **out) {
  gpudata *b = ga_hip_redux_counters(ctx);
  if (b == nullptr)
    return ga_hip_capturing(ctx) ? ga_err_set(ctx->err, GA_UNSUPPORTED_ERROR,
                                              "No counters yet and the stream records a graph: call once before recording")
                                 : ctx->err->code;
  *out = b->devptr;
  return GA_NO_ERROR;
}

// ---- checks of arguments -------------------------------------------------------

inline char *at(const GpuArray *a) { return (char *)a->data->devptr + a->offset; }
inline bool is_value(int tc) { return tc == GA_FLOAT || tc == GA_HALF || tc == GA_BFLOAT16; }

// Lowest and one past the highest byte of an array; lo == hi: no element.
void span_of(const GpuArray *a, uintptr_t *lo, uintptr_t *hi) {
  uintptr_t l = (uintptr_t)at(a), h = l + GpuArray_ITEMSIZE(a);
  for (unsigned i = 0; i < a->nd; i++) {
    if (a->dimensions[i] == 0) {
      *lo = *hi = 0;
      return;
    }
    const ssize_t far = (ssize_t)(a->dimensions[i] - 1) * a->strides[i];
    if (far < 0) l += (uintptr_t)far;
    else h += (uintptr_t)far;
  }
  *lo = l;
  *hi = h;
}

bool overlap(const GpuArray *a, const GpuArray *b) {
  uintptr_t al, ah, bl, bh;
  span_of(a, &al, &ah);
  span_of(b, &bl, &bh);
  return al < bh && bl < ah;
}

bool same_place(const GpuArray *a, const GpuArray *b) {
  if (a->nd != b->nd || at(a) != at(b) || a->typecode != b->typecode) return false;
  for (unsigned i = 0; i < a->nd; i++)
    if (a->dimensions[i] != b->dimensions[i] || (a->dimensions[i] > 1 && a->strides[i] != b->strides[i])) return false;
  return true;
}

// Whether two indices may reach one byte (dims nested by their steps never do).
bool overlaps_itself(const GpuArray *a) {
  std::vector<std::pair<size_t, size_t>> d;   // step, extent
  for (unsigned i = 0; i < a->nd; i++) {
    if (a->dimensions[i] == 0) return false;
    if (a->dimensions[i] > 1) d.emplace_back((size_t)std::llabs((long long)a->strides[i]), a->dimensions[i]);
  }
  std::sort(d.begin(), d.end());
  size_t run = GpuArray_ITEMSIZE(a);
  for (auto &e : d) {
    if (e.first < run) return true;
    run += e.first * (e.second - 1);
  }
  return false;
}

// scale * log2(e), for exponentials of 2
inline float in_powers_of_two(double scale) { return (float)((double)(float)scale * 1.4426950408889634); }

// Checks of one operator's arguments; the first failure stays.
struct argument_rules {
  gpucontext *ctx;
  const char *who;
  int err = GA_NO_ERROR;
  argument_rules(gpucontext *c, const char *w) : ctx(c), who(w) {}
  int fail(int code, const char *what) {
    if (err == GA_NO_ERROR) err = ga_err_fmt(ctx->err, code, "%s: %s", who, what);
    return err;
  }
  int fail(int code, const char *what, const char *arg) {
    if (err == GA_NO_ERROR) err = ga_err_fmt(ctx->err, code, "%s: %s: %s", who, arg, what);
    return err;
  }
  // what every array has to be
  void array(const GpuArray *a, const char *arg, unsigned nd) {
    if (err != GA_NO_ERROR) return;
    if (GpuArray_context(a) != ctx) fail(GA_INVALID_ERROR, "belongs to another context", arg);
    else if (a->nd != nd) fail(GA_INVALID_ERROR, nd == 1 ? "must have one dim" : "must have two dims", arg);
    else aligned(a, arg);
  }
  void aligned(const GpuArray *a, const char *arg) {
    if (err != GA_NO_ERROR) return;
    if (!GpuArray_ISALIGNED(a) || (uintptr_t)at(a) % gpuarray_get_type(a->typecode)->align != 0)
      fail(GA_UNALIGNED_ERROR, "not aligned", arg);
  }
  void shape(const GpuArray *a, const char *arg, size_t d0) {
    if (err == GA_NO_ERROR && a->dimensions[0] != d0) fail(GA_INVALID_ERROR, "length does not fit the others", arg);
  }
  void shape(const GpuArray *a, const char *arg, size_t d0, size_t d1) {
    if (err == GA_NO_ERROR && (a->dimensions[0] != d0 || a->dimensions[1] != d1))
      fail(GA_INVALID_ERROR, "shape does not fit the others", arg);
  }
  void rows(const GpuArray *a, const char *arg) {
    if (err == GA_NO_ERROR && a->dimensions[1] > 1 && a->strides[1] != (ssize_t)GpuArray_ITEMSIZE(a))
      fail(GA_INVALID_ERROR, "the last dim must have unit stride", arg);
  }
  void value_type(const GpuArray *a, const char *arg) {
    if (err == GA_NO_ERROR && !is_value(a->typecode))
      fail(GA_UNSUPPORTED_ERROR, "must be float, half or bfloat16", arg);
  }
  void type(const GpuArray *a, const char *arg, int tc) {
    if (err == GA_NO_ERROR && a->typecode != tc) fail(GA_VALUE_ERROR, "must be float", arg);
  }
  void id_type(const GpuArray *a, const char *arg) {
    if (err == GA_NO_ERROR && (a->typecode < GA_BYTE || a->typecode > GA_ULONG))
      fail(GA_VALUE_ERROR, "must have an integer type", arg);
  }
  // a result: writeable, nothing written twice
  void result(const GpuArray *a, const char *arg) {
    if (err != GA_NO_ERROR) return;
    if (!GpuArray_ISWRITEABLE(a)) fail(GA_VALUE_ERROR, "not writeable", arg);
    else if (overlaps_itself(a)) fail(GA_VALUE_ERROR, "overlaps itself", arg);
  }
  void apart(const GpuArray *a, const GpuArray *b, const char *arg) {
    if (err == GA_NO_ERROR && a != nullptr && b != nullptr && overlap(a, b))
      fail(GA_VALUE_ERROR, "overlaps another argument", arg);
  }
  // reading the error word waits, which a stream that records a graph does not allow
  void waits(int check_error) {
    if (err == GA_NO_ERROR && check_error && ga_hip_capturing(ctx))
      fail(GA_UNSUPPORTED_ERROR, "check_error waits, and the stream records a graph");
  }
  // a scale that a float holds
  void scale(double s) {
    if (err == GA_NO_ERROR && !std::isfinite((float)s)) fail(GA_VALUE_ERROR, "scale must be finite");
  }
  // one of exponents, above 0, which a float holds in powers of two as well
  void exponent_scale(double s) {
    if (err == GA_NO_ERROR && !((float)s > 0.0f && std::isfinite(in_powers_of_two(s))))
      fail(GA_VALUE_ERROR, "scale must be above 0, and finite when it is multiplied by log2(e)");
  }
};

// One-word errors of a kernel: the context's sticky error word, as GpuArray_take1 has it.
int lm_errbuf(gpucontext *ctx, const GpuArray *any, gpudata **errbuf) {
  (void)ctx;
  return gpudata_property(any->data, GA_CTX_PROP_ERRBUF, errbuf);
}
int lm_check_error(gpucontext *ctx, gpudata *errbuf) {
  int kerr = 0;
  int err = gpudata_read(&kerr, errbuf, 0, sizeof(int));
  if (err == GA_NO_ERROR && kerr != 0) {
    err = ga_err_set(ctx->err, GA_VALUE_ERROR, "Index out of bounds");
    kerr = 0;
    gpudata_write(errbuf, 0, &kerr, sizeof(int));
  }
  return err;
}

int no_memory(gpucontext *ctx) { return ga_err_set(ctx->err, GA_MEMORY_ERROR, "Out of memory"); }

const size_t MAX_ROWS = 0x7fffffff;   // rows or tokens that 32-bit numbers of them allow
// a launch has fewer than 2^32 lanes
inline size_t max_groups(size_t lanes) { return 0xffffffffu / lanes; }

}  // namespace

void ga_language_cache_free(gpucontext *ctx) {
  void **slot = ga_hip_language_cache_slot(ctx);
  if (*slot == nullptr) return;
  lm_cache *cache = (lm_cache *)*slot;
  *slot = nullptr;
  for (auto &kv : *cache) GpuKernel_clear(&kv.second);
  delete cache;
}

// The kernel text of a variant (packed as lm_variant::key packs it), as a
// malloc'd string; behind the "hip_language_source" hook.
char *ga_language_gen_source(unsigned long long variant) {
  try {
    return strdup(lm_source(lm_variant(variant)).c_str());
  } catch (...) {
    return nullptr;
  }
}

// ---- embedding -----------------------------------------------------------------

static int embedding(GpuArray *out, const GpuArray *table, const GpuArray *ids, double scale, ssize_t ignore,
                     int check_error) {
  gpucontext *ctx = GpuArray_context(out);
  argument_rules c(ctx, "embedding");
  c.array(out, "out", 2);
  c.array(table, "table", 2);
  c.array(ids, "ids", 1);
  if (c.err != GA_NO_ERROR) return c.err;
  const size_t n = ids->dimensions[0], v = table->dimensions[0], d = table->dimensions[1];
  c.shape(out, "out", n, d);
  c.value_type(out, "out");
  c.value_type(table, "table");
  c.id_type(ids, "ids");
  c.rows(out, "out");
  c.rows(table, "table");
  c.result(out, "out");
  c.apart(out, table, "out");
  c.apart(out, ids, "out");
  c.scale(scale);
  c.waits(check_error);
  if (c.err != GA_NO_ERROR) return c.err;
  if (n == 0 || d == 0) return GA_NO_ERROR;
  // lanes of a row: a power of two, each with 16 bytes of the result; a lane moves four rows
  const size_t lane_cols = 16 / gpuarray_get_elsize(out->typecode);
  const size_t row_lanes = (d + lane_cols - 1) / lane_cols, segments = (row_lanes + 255) / 256;
  unsigned lanes_log2 = 0;
  while (lanes_log2 < 8 && ((size_t)1 << lanes_log2) < row_lanes) lanes_log2++;
  const size_t row_groups = (n + ((size_t)1024 >> lanes_log2) - 1) / ((size_t)1024 >> lanes_log2);
  if (row_groups > max_groups(256) || segments > max_groups(256) / row_groups)
    return c.fail(GA_XLARGE_ERROR, "too many elements");
  GpuKernel *k;
  gpudata *errbuf = nullptr;
  int err = lm_kernel(ctx, lm_variant(LM_EMBED, table->typecode, out->typecode, ids->typecode, 0), "lm_embed_rows",
                      sizeof(embed_args), &k);
  if (err == GA_NO_ERROR) err = lm_errbuf(ctx, out, &errbuf);
  if (err != GA_NO_ERROR) return err;
  embed_args a = {at(out), at(table), at(ids), errbuf->devptr, out->strides[0], table->strides[0], ids->strides[0],
                  (int64_t)n, (int64_t)v, (int64_t)d, ignore, (float)scale, lanes_log2, (uint32_t)segments};
  err = lm_launch(k, row_groups * segments, 256, &a);
  return err == GA_NO_ERROR && check_error ? lm_check_error(ctx, errbuf) : err;
}

static int embedding_grad(GpuArray *grad, const GpuArray *dout, const GpuArray *ids, double scale, ssize_t ignore,
                          int accumulate, int check_error) {
  gpucontext *ctx = GpuArray_context(grad);
  argument_rules c(ctx, "embedding_grad");
  c.array(grad, "grad", 2);
  c.array(dout, "dout", 2);
  c.array(ids, "ids", 1);
  if (c.err != GA_NO_ERROR) return c.err;
  const size_t n = ids->dimensions[0], v = grad->dimensions[0], d = grad->dimensions[1];
  c.shape(dout, "dout", n, d);
  c.value_type(grad, "grad");
  c.value_type(dout, "dout");
  c.id_type(ids, "ids");
  c.rows(grad, "grad");
  c.rows(dout, "dout");
  c.result(grad, "grad");
  c.apart(grad, dout, "grad");
  c.apart(grad, ids, "grad");
  c.scale(scale);
  c.waits(check_error);
  if (c.err != GA_NO_ERROR) return c.err;
  if (d == 0 || (v == 0 && n == 0)) return GA_NO_ERROR;
  if (v > MAX_ROWS || n > MAX_ROWS) return c.fail(GA_XLARGE_ERROR, "too many rows");

  const size_t osize = gpuarray_get_elsize(grad->typecode);
  const size_t cols = 64 * 16 / std::max(osize, gpuarray_get_elsize(dout->typecode));   // of a wavefront
  const size_t tiles = (d + cols - 1) / cols;
  // rows that half a wavefront covers: several chunks of tokens side by side in one
  // (65536 tokens of 64 bfloat16 added to floats 41 us, with a wavefront a chunk
  // 50; of 120 45 and 50; a million of 16 101 and 122)
  unsigned lanes_log2 = 3;
  while (((size_t)cols / 64 << lanes_log2) < d && lanes_log2 < 6) lanes_log2++;
  const bool narrow = lanes_log2 < 6, dense = v <= 1 || grad->strides[0] == (ssize_t)(d * osize);
  const lm_variant vg(LM_EMBED_GRAD, dout->typecode, grad->typecode, ids->typecode, narrow);
  gpudata *errbuf = nullptr;
  embed_grad_args a = {at(grad), at(dout), nullptr, nullptr, nullptr, at(ids), nullptr, ids->strides[0], ignore,
                       grad->strides[0], dout->strides[0], (int64_t)v, (int64_t)d, (float)scale, accumulate != 0,
                       (uint32_t)n, 0, 0, (uint32_t)tiles, 0, lanes_log2, dense, 0};
  int err = lm_errbuf(ctx, grad, &errbuf);
  if (err != GA_NO_ERROR) return err;
  a.err = errbuf->devptr;
  // Up to 256 tokens, as many as a group has lanes, are not sorted (256 of 1024 bfloat16 into
  // 50257 rows of floats that are cleared 33 us, sorted 46; into 1000 rows of 256 5 and 13; added 5.5 and 16).
  if (n <= 256) {
    GpuKernel *kfew = nullptr;
    err = lm_kernel(ctx, vg, "lm_embed_grad_few", sizeof(embed_grad_args), &kfew);
    // A group has four tiles of columns, one for each wavefront, and 8 KiB of rows
    // (zeroing 50257 rows of 1024 floats for 256 tokens, by 4, 8, 16 KiB: 49, 32, 38 us).
    // Many rows that do not begin on 16-byte boundaries are taken whole, so that they are
    // zeroed end to end (22000 rows of 4413 bfloat16: 44 us, in parts 56; but 1000
    // rows of 6000 floats 17.5 us, in parts 10.5).
    a.part_tiles = !accumulate && dense && d * osize % 16 != 0 && tiles <= 16 && v >= 4096 ? 16 : 4;
    const size_t parts = (tiles + a.part_tiles - 1) / a.part_tiles;
    const size_t fit = std::max<size_t>(8192 / (std::min(d, a.part_tiles * cols) * osize), 1);
    a.rows = (uint32_t)std::min({fit, v * parts / 512 + 1, (size_t)512});
    const size_t row_groups = accumulate ? n : v ? (v + a.rows - 1) / a.rows : 1;
    if (row_groups == 0) return GA_NO_ERROR;
    if (parts > max_groups(256) / row_groups) return c.fail(GA_XLARGE_ERROR, "too many elements");
    if (err == GA_NO_ERROR) err = lm_launch(kfew, row_groups * parts, 256, &a);
    return err == GA_NO_ERROR && check_error ? lm_check_error(ctx, errbuf) : err;
  }
  // Tokens of a chunk: enough chunks to fill the chip with wavefronts, and
  // not so few tokens that partial sums (two rows a chunk at most) count, nor
  // the parts of a token that comes very often (65536 tokens of 2048 added, by the least number of wavefronts:
  // 2048 185 us, 4096 138, 8192 128, 16384 132).
  const size_t per_wave = narrow ? (size_t)64 >> lanes_log2 : 1;   // chunks
  size_t chunk = 8;
  while (chunk < 256 && n / (chunk * 2) / per_wave * tiles >= (narrow ? 2048u : 8192u)) chunk *= 2;
  const size_t chunks = (n + chunk - 1) / chunk;
  if (tiles > max_groups(256) / chunks) return c.fail(GA_XLARGE_ERROR, "too many elements");
  // The digits: as few passes as ten bits a digit allow.
  unsigned bits = 1;
  while (v >> bits != 0) bits++;
  const unsigned passes = (bits + 9) / 10;
  bits = (bits + passes - 1) / passes;
  // Up to 8192 tokens, 8 a lane, one group sorts by itself, up to 16384 where clearing the
  // rows takes longer than that; more are sorted by many, with few tokens a lane while there are
  // few groups.  Kernel time of the sort of ids below 50257, us:
  //   tokens                   4097    8192    8193   16384
  //   one group                18.3    19.2    35.1    39.6
  //   many                     21.1    23.0    23.2    20.0
  //   tokens                  65536  250000  500000 1000000 1200000
  //   one a lane                 24      32      40      65      79
  //   two                        26      37      37      50      65
  //   four                       30      41      48      48      62
  const size_t clear_bytes = accumulate ? 0 : v * d * osize;
  const bool small = n <= 8192 || (n <= 16384 && clear_bytes / n >= 14000);
  const size_t per_lane = small ? (n + 1023) / 1024 : n <= ((size_t)1 << 18) ? 1 : n <= ((size_t)1 << 20) ? 2 : 4;
  unsigned items = 1;
  while (items < per_lane) items *= 2;
  const size_t groups = small ? 1 : (n + 1024 * items - 1) / (1024 * items);
  // Where there are few counts every group of lm_sort_move adds them up itself
  // (10000 tokens, 50257 rows of 64 floats: 34 us, with a launch for that 39; past 32768 it is no faster).
  const bool direct = groups << bits <= 32768;

  // scratch: two sets of keys and places, the counts of the digits, the partial sums
  const size_t list = (n * 4 + 255) & ~(size_t)255;
  const size_t counts = small ? 0 : (((groups + 1) << bits) * 4 + 255) & ~(size_t)255;
  const size_t partials = chunks * 2 * tiles * cols * 4;
  char *scratch = nullptr;
  GpuKernel *ksmall = nullptr, *kcount = nullptr, *kscan = nullptr, *kmove = nullptr, *ksum = nullptr, *kjoin = nullptr;
  const lm_variant vs(LM_SORT, GA_FLOAT, GA_FLOAT, ids->typecode, items);
  if (small) {
    err = lm_kernel(ctx, vs, "lm_sort_small", sizeof(sorting_args), &ksmall);
  } else {
    err = lm_kernel(ctx, vs, "lm_sort_count", sizeof(sorting_args), &kcount);
    if (err == GA_NO_ERROR && !direct) err = lm_kernel(ctx, vs, "lm_sort_scan", sizeof(sorting_args), &kscan);
    if (err == GA_NO_ERROR) err = lm_kernel(ctx, vs, "lm_sort_move", sizeof(sorting_args), &kmove);
  }
  if (err == GA_NO_ERROR) err = lm_kernel(ctx, vg, "lm_embed_grad_sum", sizeof(embed_grad_args), &ksum);
  if (err == GA_NO_ERROR) err = lm_kernel(ctx, vg, "lm_embed_grad_join", sizeof(embed_grad_args), &kjoin);
  if (err == GA_NO_ERROR) err = lm_scratch(ctx, 4 * list + counts + partials + 256, &scratch);
  if (err != GA_NO_ERROR) return err;

  char *lists[4] = {scratch, scratch + list, scratch + 2 * list, scratch + 3 * list};
  sorting_args s;
  memset(&s, 0, sizeof(s));
  s.ids = at(ids);
  s.id_step = ids->strides[0];
  s.err = errbuf->devptr;
  s.counts = scratch + 4 * list;
  s.ignore = ignore;
  s.v = (int64_t)v;
  s.n = (uint32_t)n;
  s.groups = (uint32_t)groups;
  s.bits = bits;
  s.passes = passes;
  s.direct = direct;
  // rows to clear, as one where they lie end to end
  size_t units = 0;
  if (!accumulate && v > 0) {
    s.fill = at(grad);
    s.fill_rows = dense ? 1 : (int64_t)v;
    s.fill_row = grad->strides[0];
    s.fill_bytes = (int64_t)(dense ? v * d * osize : d * osize);
    units = (size_t)s.fill_rows * (((size_t)s.fill_bytes + 16383) / 16384);
  }
  // launches of the sort that clear a share each, with up to 1024 groups more for it
  const size_t launches = small ? 1 : (direct ? 2 : 3) * passes;
  size_t launched = 0;
  auto sort_launch = [&](GpuKernel *k, size_t busy) -> int {
    s.fill_unit0 = (int64_t)(units * launched / launches);
    s.fill_unit1 = (int64_t)(units * (launched + 1) / launches);
    launched++;
    const size_t more = std::min<size_t>(((size_t)(s.fill_unit1 - s.fill_unit0) + 15) / 16, 1024);
    return lm_launch(k, busy + more, 1024, &s);
  };
  if (small) {
    s.key = lists[0];
    s.order = lists[1];
    err = sort_launch(ksmall, 1);
  } else {
    for (unsigned pass = 0; pass < passes && err == GA_NO_ERROR; pass++) {
      const int from = pass & 1 ? 0 : 2, to = 2 - from;
      s.shift = pass * bits;
      s.key_in = lists[from];
      s.order_in = lists[from + 1];
      s.key = lists[to];
      s.order = lists[to + 1];
      err = sort_launch(kcount, groups);
      if (err == GA_NO_ERROR && !direct) err = sort_launch(kscan, (((size_t)1 << bits) + 15) / 16);
      if (err == GA_NO_ERROR) err = sort_launch(kmove, groups);
    }
  }
  if (err == GA_NO_ERROR && n > 0) {
    a.key = s.key;
    a.order = s.order;
    a.partials = scratch + 4 * list + counts;
    a.chunk = (uint32_t)chunk;
    a.chunks = (uint32_t)chunks;
    err = lm_launch(ksum, (chunks * tiles + 4 * per_wave - 1) / (4 * per_wave), 256, &a);
    if (err == GA_NO_ERROR && chunks > 1) err = lm_launch(kjoin, chunks * tiles, 256, &a);
  }
  return err == GA_NO_ERROR && check_error ? lm_check_error(ctx, errbuf) : err;
}

// ---- log probabilities -----------------------------------------------------------

static int token_logprobs(GpuArray *logp, GpuArray *entropy, GpuArray *stats, GpuArray *top_logp, GpuArray *top_ids,
                          const GpuArray *logits, const GpuArray *ids, double scale, ssize_t ignore, int check_error) {
  gpucontext *ctx = GpuArray_context(logits);
  argument_rules c(ctx, "token_logprobs");
  c.array(logits, "logits", 2);
  if (c.err != GA_NO_ERROR) return c.err;
  const size_t t = logits->dimensions[0], v = logits->dimensions[1];
  c.value_type(logits, "logits");
  c.rows(logits, "logits");
  if ((logp == nullptr) != (ids == nullptr)) return c.fail(GA_VALUE_ERROR, "logp and ids go together");
  if ((top_logp == nullptr) != (top_ids == nullptr)) return c.fail(GA_VALUE_ERROR, "top_logp and top_ids go together");
  if (ids != nullptr) {
    c.array(ids, "ids", 1);
    c.id_type(ids, "ids");
    c.shape(ids, "ids", t);
  }
  GpuArray *const results[5] = {logp, entropy, stats, top_logp, top_ids};
  const char *const names[5] = {"logp", "entropy", "stats", "top_logp", "top_ids"};
  for (int i = 0; i < 5; i++) {
    if (results[i] == nullptr) continue;
    c.array(results[i], names[i], i < 2 ? 1 : 2);
    if (c.err != GA_NO_ERROR) return c.err;
    if (i < 2) c.shape(results[i], names[i], t);
    else if (i == 2) c.shape(stats, names[i], t, 2);
    else c.shape(results[i], names[i], t, top_ids->nd == 2 ? top_ids->dimensions[1] : 0);
    if (i < 4) c.type(results[i], names[i], GA_FLOAT);
    else if (top_ids->typecode != GA_INT && top_ids->typecode != GA_LONG)
      c.fail(GA_VALUE_ERROR, "must be int or long", names[i]);
    c.result(results[i], names[i]);
    c.apart(results[i], logits, names[i]);
    c.apart(results[i], ids, names[i]);
    for (int j = 0; j < i; j++) c.apart(results[i], results[j], names[i]);
  }
  c.exponent_scale(scale);
  c.waits(check_error);
  if (c.err != GA_NO_ERROR) return c.err;
  const size_t top = top_ids ? top_ids->dimensions[1] : 0;
  if (top > GA_TOKEN_LOGPROBS_MAX_TOP || top > v)
    return c.fail(GA_VALUE_ERROR, "more alternatives than the vocabulary or GA_TOKEN_LOGPROBS_MAX_TOP has");
  if (t == 0 || (logp == nullptr && entropy == nullptr && stats == nullptr && top == 0)) return GA_NO_ERROR;
  if (v == 0) return c.fail(GA_VALUE_ERROR, "empty vocabulary");
  if (v > 0x3fffffff) return c.fail(GA_XLARGE_ERROR, "too many columns");
  // A row that a wavefront covers in eight rounds of loads belongs to one
  // wavefront, a longer one to a group, which grows while there are too few
  // rows to fill the chip; below that, rows are cut in pieces of at least one
  // batch for each lane, of which the last one to end joins them all.  Rows of bfloat16 with
  // entropy, us by the lanes 64, 256, 512, 1024 (and pieces):
  //   32768 rows of 2000     32    59   139   331
  //   32768 rows of 4000     51    68   134   324
  //   4096 rows of 50257     68    68    73   101
  //   512 rows of 50257      32    15    13    15
  //   128 rows of 50257      30    11     7.9   7.8   (8.4)
  //   8 rows of 50257        29     9.2   6.9   6.8   (5.6)
  const size_t row_chunks = v * gpuarray_get_elsize(logits->typecode) / 16 + 1;
  const size_t cus = ga_hip_numprocs(ctx) ? ga_hip_numprocs(ctx) : 256;
  unsigned lanes = 64;
  if (row_chunks > 512) {
    lanes = 256;
    while (lanes < 1024 && t * lanes < cus * 1024 && row_chunks > 8 * lanes) lanes *= 2;
  }
  size_t pieces = 1, piece_chunks = row_chunks;
  if (row_chunks > 512 && t * 2 <= cus && t <= ga_hip_redux_counters_max) {
    lanes = 256;
    // (one batch of loads: 16 elements a lane; half of that or twice as much: 8 rows of 50257 floats,
    // 20 alternatives, 11.8, 10.4 and 11.4 us, of bfloat16 11.6, 10.2 and 11.3)
    const size_t batch = 256 * gpuarray_get_elsize(logits->typecode);
    pieces = std::min((2 * cus + t - 1) / t, (row_chunks + batch - 1) / batch);
    piece_chunks = (row_chunks + pieces - 1) / pieces;
    pieces = (row_chunks + piece_chunks - 1) / piece_chunks;
  }
  const bool split = pieces > 1;
  const size_t groups = split ? t * pieces : lanes < 256 ? (t + 3) / 4 : t;
  if (groups > max_groups(std::max(lanes, 256u))) return c.fail(GA_XLARGE_ERROR, "too many rows");
  const size_t partial_bytes = 16 + 8 * top;
  const lm_variant var(LM_LOGPROBS, logits->typecode, GA_FLOAT, ids ? ids->typecode : GA_INT,
                       logprobs_extra(lanes, entropy != nullptr, top != 0, split));
  GpuKernel *k;
  gpudata *errbuf = nullptr;
  char *scratch = nullptr;
  void *counters = nullptr;   // the last piece of a row joins them
  int err = lm_kernel(ctx, var, "lm_logprobs_rows", sizeof(logprobs_args), &k);
  if (err == GA_NO_ERROR && split) err = lm_counters(ctx, &counters);
  if (err == GA_NO_ERROR && split) err = lm_scratch(ctx, t * pieces * partial_bytes, &scratch);
  if (err == GA_NO_ERROR) err = lm_errbuf(ctx, logits, &errbuf);
  if (err != GA_NO_ERROR) return err;
  auto ptr = [](const GpuArray *x) -> void * { return x ? at(x) : nullptr; };
  auto step = [](const GpuArray *x, unsigned i) -> int64_t { return x ? x->strides[i] : 0; };
  logprobs_args a = {at(logits), ptr(ids), ptr(logp), ptr(entropy), ptr(stats), ptr(top_logp), ptr(top_ids),
                     errbuf->devptr, scratch, logits->strides[0], step(ids, 0), step(logp, 0), step(entropy, 0),
                     step(stats, 0), step(stats, 1), step(top_logp, 0), step(top_logp, 1), step(top_ids, 0),
                     step(top_ids, 1), (int64_t)t, (int64_t)v, ignore, (float)scale,
                     in_powers_of_two(scale), (int32_t)top,
                     top_ids != nullptr && top_ids->typecode == GA_LONG, (uint32_t)pieces, (uint32_t)piece_chunks,
                     (uint32_t)partial_bytes, 0, counters};
  err = lm_launch(k, groups, std::max(lanes, 256u), &a);
  return err == GA_NO_ERROR && check_error ? lm_check_error(ctx, errbuf) : err;
}

static int token_logprobs_grad(GpuArray *dlogits, const GpuArray *logits, const GpuArray *ids, const GpuArray *stats,
                               const GpuArray *dlogp, const GpuArray *entropy, const GpuArray *dentropy, double scale,
                               ssize_t ignore, int check_error) {
  gpucontext *ctx = GpuArray_context(dlogits);
  argument_rules c(ctx, "token_logprobs_grad");
  c.array(dlogits, "dlogits", 2);
  c.array(logits, "logits", 2);
  c.array(stats, "stats", 2);
  if (c.err != GA_NO_ERROR) return c.err;
  const size_t t = logits->dimensions[0], v = logits->dimensions[1];
  c.shape(dlogits, "dlogits", t, v);
  c.shape(stats, "stats", t, 2);
  c.value_type(logits, "logits");
  if (c.err == GA_NO_ERROR && dlogits->typecode != logits->typecode)
    c.fail(GA_VALUE_ERROR, "must have the type of logits", "dlogits");
  c.type(stats, "stats", GA_FLOAT);
  c.rows(dlogits, "dlogits");
  c.rows(logits, "logits");
  c.result(dlogits, "dlogits");
  if ((ids == nullptr) != (dlogp == nullptr)) return c.fail(GA_VALUE_ERROR, "ids and dlogp go together");
  if ((entropy == nullptr) != (dentropy == nullptr)) return c.fail(GA_VALUE_ERROR, "entropy and dentropy go together");
  const GpuArray *const vectors[4] = {ids, dlogp, entropy, dentropy};
  const char *const names[4] = {"ids", "dlogp", "entropy", "dentropy"};
  for (int i = 0; i < 4; i++) {
    if (vectors[i] == nullptr) continue;
    c.array(vectors[i], names[i], 1);
    if (c.err != GA_NO_ERROR) return c.err;
    c.shape(vectors[i], names[i], t);
    if (i == 0) c.id_type(ids, names[i]);
    else c.type(vectors[i], names[i], GA_FLOAT);
    c.apart(dlogits, vectors[i], "dlogits");
  }
  c.apart(dlogits, stats, "dlogits");
  if (c.err == GA_NO_ERROR && !same_place(dlogits, logits)) c.apart(dlogits, logits, "dlogits");
  c.exponent_scale(scale);
  c.waits(check_error);
  if (c.err != GA_NO_ERROR) return c.err;
  if (t == 0 || v == 0) return GA_NO_ERROR;
  if (v > 0x3fffffff) return c.fail(GA_XLARGE_ERROR, "too many columns");
  // a wavefront's share of a row: 32 elements a lane (and one chunk more, for rows that start inside one)
  const size_t esize = gpuarray_get_elsize(logits->typecode);
  const size_t segments = (v * esize / 16 + 2 + 128 * esize - 1) / (128 * esize);
  if (segments > 4 * max_groups(256) / t) return c.fail(GA_XLARGE_ERROR, "too many elements");
  GpuKernel *k;
  gpudata *errbuf = nullptr;
  const lm_variant var(LM_LOGPROBS_GRAD, logits->typecode, GA_FLOAT, ids ? ids->typecode : GA_INT, entropy != nullptr);
  int err = lm_kernel(ctx, var, "lm_logprobs_grad_rows", sizeof(logprobs_grad_args), &k);
  if (err == GA_NO_ERROR) err = lm_errbuf(ctx, logits, &errbuf);
  if (err != GA_NO_ERROR) return err;
  auto ptr = [](const GpuArray *x) -> void * { return x ? at(x) : nullptr; };
  auto step = [](const GpuArray *x, unsigned i) -> int64_t { return x ? x->strides[i] : 0; };
  logprobs_grad_args a = {at(dlogits), at(logits), ptr(ids), at(stats), ptr(dlogp), ptr(entropy), ptr(dentropy),
                          errbuf->devptr, dlogits->strides[0], logits->strides[0], step(ids, 0), stats->strides[0],
                          stats->strides[1], step(dlogp, 0), step(entropy, 0), step(dentropy, 0), (int64_t)t,
                          (int64_t)v, ignore, (float)scale, in_powers_of_two(scale),
                          (uint32_t)segments};
  err = lm_launch(k, (t * segments + 3) / 4, 256, &a);
  return err == GA_NO_ERROR && check_error ? lm_check_error(ctx, errbuf) : err;
}

// ---- global norm -------------------------------------------------------------------

// What a call works on: arrays with at least one element, in pieces.
struct norm_plan {
  std::vector<tensor_arg> tensors;
  bool doubles = false;   // whose squares may leave the range of a double
};

// Pieces of 16 KiB: four chunks for each lane of a group, loaded at once.
// Clipping 600 MB of bfloat16, by the piece: 16 KiB 186 us, 32 KiB 198, 64 KiB
// 213.  The norm's groups, one for each compute unit, take a range of them each
// (600 MB in 256 to 2048 groups: 107 to 109 us), so that the last one of them can
// finish the norm.
static const size_t NORM_PIECE = 1024;       // chunks of 16 bytes
static const size_t NORM_MAX_GROUPS = 256;   // per table

static int norm_check(argument_rules &c, const GpuArray *norm) {
  if (norm == nullptr) return c.err;
  if (norm->nd > 1 || (norm->nd == 1 && norm->dimensions[0] != 1))
    return c.fail(GA_INVALID_ERROR, "must be 0-d or have one element", "norm");
  if (norm->typecode != GA_FLOAT && norm->typecode != GA_DOUBLE)
    return c.fail(GA_VALUE_ERROR, "must be float or double", "norm");
  if (GpuArray_context(norm) != c.ctx) return c.fail(GA_INVALID_ERROR, "the arrays belong to different contexts");
  c.aligned(norm, "norm");
  c.result(norm, "norm");
  return c.err;
}

// The arrays `as` and, if rs is not NULL, what clipping writes, checked against each other.
static int norm_arrays(argument_rules &c, GpuArray **rs, const GpuArray **as, size_t n, norm_plan *plan) {
  std::vector<std::pair<uintptr_t, uintptr_t>> written, read;
  plan->tensors.reserve(n);
  for (size_t i = 0; i < n; i++) {
    const GpuArray *a = as[i], *r = rs != nullptr ? rs[i] : a;
    if (GpuArray_context(a) != c.ctx) return c.fail(GA_INVALID_ERROR, "the arrays belong to different contexts");
    if (!is_value(a->typecode) && a->typecode != GA_DOUBLE)
      return c.fail(GA_UNSUPPORTED_ERROR, "arrays must be float, half, bfloat16 or double");
    if (!GpuArray_ISONESEGMENT(a)) return c.fail(GA_INVALID_ERROR, "arrays must be contiguous");
    c.aligned(a, "arrays");
    if (c.err != GA_NO_ERROR) return c.err;
    size_t count = 1;
    for (unsigned j = 0; j < a->nd; j++) count *= a->dimensions[j];
    const size_t size = GpuArray_ITEMSIZE(a);
    if (rs != nullptr) {
      if (r != a && !same_place(r, a)) {
        if (GpuArray_context(r) != c.ctx) return c.fail(GA_INVALID_ERROR, "the arrays belong to different contexts");
        if (r->nd != a->nd || r->typecode != a->typecode)
          return c.fail(GA_INVALID_ERROR, "a result differs from its array in shape or type");
        for (unsigned j = 0; j < a->nd; j++)
          if (r->dimensions[j] != a->dimensions[j] || (a->dimensions[j] > 1 && count > 0 && r->strides[j] != a->strides[j]))
            return c.fail(GA_INVALID_ERROR, "a result differs from its array in shape or strides");
        c.aligned(r, "results");
        if (count > 0) read.emplace_back((uintptr_t)at(a), (uintptr_t)at(a) + count * size);
      }
      if (!GpuArray_ISWRITEABLE(r)) return c.fail(GA_VALUE_ERROR, "a result is not writeable");
      if (c.err != GA_NO_ERROR) return c.err;
      if (count > 0) written.emplace_back((uintptr_t)at(r), (uintptr_t)at(r) + count * size);
    }
    if (count == 0) continue;
    const uint64_t per = NORM_PIECE * (16 / size), p = (count + per - 1) / per;
    if (p > max_groups(256)) return c.fail(GA_XLARGE_ERROR, "an array is too large");
    tensor_arg t = {at(a), at(r), (int64_t)count, (uint32_t)p,   // (`first` holds the count of pieces until a table is made)
                    a->typecode == GA_FLOAT ? 0u : a->typecode == GA_HALF ? 1u : a->typecode == GA_BFLOAT16 ? 2u : 3u};
    plan->tensors.push_back(t);
    plan->doubles |= a->typecode == GA_DOUBLE;
  }
  // no two results overlap, and none overlaps an operand that is not itself
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); i++)
    if (written[i].first < written[i - 1].second) return c.fail(GA_VALUE_ERROR, "results overlap");
  for (auto &x : read) {
    auto it = std::lower_bound(written.begin(), written.end(), std::make_pair(x.second, (uintptr_t)0));
    if (it != written.begin() && (it - 1)->second > x.first)
      return c.fail(GA_VALUE_ERROR, "a result overlaps another array");
  }
  return GA_NO_ERROR;
}

// `norm` must lie outside all the arrays.
static int norm_apart(argument_rules &c, const norm_plan &plan, const GpuArray *norm) {
  if (norm == nullptr) return GA_NO_ERROR;
  const uintptr_t lo = (uintptr_t)at(norm), hi = lo + GpuArray_ITEMSIZE(norm);
  static const size_t sizes[4] = {4, 2, 2, 8};
  for (const tensor_arg &t : plan.tensors) {
    const size_t bytes = (size_t)t.count * sizes[t.type];
    if ((lo < (uintptr_t)t.in + bytes && (uintptr_t)t.in < hi) || (lo < (uintptr_t)t.out + bytes && (uintptr_t)t.out < hi))
      return c.fail(GA_VALUE_ERROR, "overlaps an array", "norm");
  }
  return GA_NO_ERROR;
}

// Launches on tables: of a list of arrays cut into argument lists, or one in
// device memory.  There is one at least, with no arrays if need be.
struct norm_table {
  const tensor_arg *tensors;   // NULL: in device memory
  const void *device;
  uint32_t n, pieces;
};
static int norm_run(argument_rules &c, const std::vector<norm_table> &tables, bool doubles, bool clip, double max_norm,
                    const GpuArray *norm) {
  gpucontext *ctx = c.ctx;
  const bool by_table = tables.size() == 1 && tables[0].tensors == nullptr;
  const size_t size = by_table ? sizeof(table_args) : sizeof(tensors_args);
  const lm_variant vn(LM_NORM, GA_FLOAT, GA_FLOAT, GA_INT, by_table | (doubles ? 2u : 0u)), vc(LM_CLIP, GA_FLOAT, GA_FLOAT, GA_INT, by_table);
  char *scratch = nullptr;
  void *counters = nullptr;
  GpuKernel *kpieces = nullptr, *kclip = nullptr;
  int err = lm_kernel(ctx, vn, "lm_norm_pieces", size, &kpieces);
  if (err == GA_NO_ERROR && clip) err = lm_kernel(ctx, vc, "lm_clip_pieces", size, &kclip);
  if (err == GA_NO_ERROR) err = lm_counters(ctx, &counters);
  // partial sums: of the squares, and where there are doubles of the large and of the small ones behind them
  const size_t partials = tables.size() * NORM_MAX_GROUPS;
  if (err == GA_NO_ERROR) err = lm_scratch(ctx, 256 + (doubles ? 3 : 1) * partials * sizeof(double), &scratch);
  if (err != GA_NO_ERROR) return err;

  tensors_args args;
  table_args *const short_args = (table_args *)&args;
  memset(&args, 0, sizeof(args));
  norm_args &a = args.a;
  a.result = scratch;
  a.partials = scratch + 256;
  a.norm = norm ? at(norm) : nullptr;
  a.norm_double = norm != nullptr && norm->typecode == GA_DOUBLE;
  a.max_norm = max_norm;
  a.piece = (uint32_t)NORM_PIECE;
  a.ends = doubles ? (uint32_t)partials : 0;
  auto take = [&](const norm_table &t) {
    a.n = t.n;
    a.pieces = t.pieces;
    if (t.tensors != nullptr) memcpy(args.tensors, t.tensors, t.n * sizeof(tensor_arg));
    else short_args->tensors = t.device;
  };
  // the last table's groups count themselves in, and the last of those finishes the norm
  for (size_t i = 0; i < tables.size() && err == GA_NO_ERROR; i++) {
    take(tables[i]);
    const size_t groups = std::min<size_t>(std::max(a.pieces, 1u), NORM_MAX_GROUPS);
    a.partial0 = a.npartials;
    a.npartials += (uint32_t)groups;
    a.counter = i + 1 == tables.size() ? counters : nullptr;
    err = lm_launch(kpieces, groups, 256, &args);
  }
  for (size_t i = 0; i < tables.size() && err == GA_NO_ERROR && clip; i++) {
    if (tables.size() > 1) take(tables[i]);
    if (a.pieces != 0) err = lm_launch(kclip, a.pieces, 256, &args);
  }
  return err;
}

// One call on a list of arrays, which travel with the arguments of the launches.
static int norm_and_clip(GpuArray **rs, const GpuArray **as, size_t n, double max_norm, GpuArray *norm, const char *who) {
  if (n == 0 && norm == nullptr) return GA_NO_ERROR;
  argument_rules c(GpuArray_context(norm != nullptr ? norm : as[0]), who);
  norm_plan plan;
  if (std::isnan(max_norm) || max_norm < 0) return c.fail(GA_VALUE_ERROR, "max_norm must be 0 or above");
  if (norm_check(c, norm) != GA_NO_ERROR || norm_arrays(c, rs, as, n, &plan) != GA_NO_ERROR ||
      norm_apart(c, plan, norm) != GA_NO_ERROR)
    return c.err;
  std::vector<norm_table> tables;
  for (size_t i = 0; i < plan.tensors.size(); i++) {
    const uint32_t p = plan.tensors[i].first;
    if (tables.empty() || tables.back().n == LM_TENSORS || tables.back().pieces + (uint64_t)p > max_groups(256))
      tables.push_back({&plan.tensors[i], nullptr, 0, 0});
    plan.tensors[i].first = tables.back().pieces;
    tables.back().n++;
    tables.back().pieces += p;
  }
  if (tables.empty()) tables.push_back({nullptr, nullptr, 0, 0});
  return norm_run(c, tables, plan.doubles, rs != nullptr, max_norm, norm);
}

struct _GpuGlobalNorm {
  gpucontext *ctx;
  norm_plan plan;
  bool clips;
  gpudata *table;
  uint32_t pieces;
  std::vector<gpudata *> held;   // the arrays' buffers
};

static int global_norm_new(GpuGlobalNorm **out, gpucontext *ctx, const GpuArray **as, GpuArray **rs, size_t n) {
  argument_rules c(ctx, "GpuGlobalNorm_new");
  if (ga_hip_capturing(ctx))
    return c.fail(GA_UNSUPPORTED_ERROR, "the stream records a graph: make the operator before recording");
  std::unique_ptr<GpuGlobalNorm> g(new GpuGlobalNorm());
  g->ctx = ctx;
  g->clips = rs != nullptr;
  g->table = nullptr;
  if (norm_arrays(c, rs, as, n, &g->plan) != GA_NO_ERROR) return c.err;
  uint64_t pieces = 0;
  for (tensor_arg &t : g->plan.tensors) {
    const uint32_t p = t.first;
    t.first = (uint32_t)pieces;
    pieces += p;
    if (pieces > max_groups(256)) return c.fail(GA_XLARGE_ERROR, "the arrays are too large together");
  }
  g->pieces = (uint32_t)pieces;
  g->held.reserve(2 * n);
  if (!g->plan.tensors.empty()) {
    int err = GA_NO_ERROR;
    g->table = gpudata_alloc(ctx, g->plan.tensors.size() * sizeof(tensor_arg), g->plan.tensors.data(), GA_BUFFER_INIT, &err);
    if (g->table == nullptr) return err;
  }
  for (size_t i = 0; i < n; i++) {
    g->held.push_back(as[i]->data);
    if (rs != nullptr) g->held.push_back(rs[i]->data);
  }
  for (gpudata *b : g->held) gpudata_retain(b);
  *out = g.release();
  return GA_NO_ERROR;
}

static int global_norm_call(const GpuGlobalNorm *g, bool clip, double max_norm, GpuArray *norm, const char *who) {
  argument_rules c(g->ctx, who);
  if (std::isnan(max_norm) || max_norm < 0) return c.fail(GA_VALUE_ERROR, "max_norm must be 0 or above");
  if (clip && !g->clips) return c.fail(GA_INVALID_ERROR, "the operator was made without results");
  if (norm_check(c, norm) != GA_NO_ERROR || norm_apart(c, g->plan, norm) != GA_NO_ERROR) return c.err;
  if (g->table == nullptr && norm == nullptr) return GA_NO_ERROR;
  const std::vector<norm_table> tables = {
      {nullptr, g->table ? g->table->devptr : nullptr, (uint32_t)g->plan.tensors.size(), g->pieces}};
  return norm_run(c, tables, g->plan.doubles, clip, max_norm, norm);
}

// ---- the C entry points: nothing thrown leaves them ----------------------------------

extern "C" {

int GpuArray_embedding(GpuArray *out, const GpuArray *table, const GpuArray *ids, double scale, ssize_t ignore,
                       int check_error) {
  try {
    return embedding(out, table, ids, scale, ignore, check_error);
  } catch (...) {   // (std::bad_alloc, std::length_error)
    return no_memory(GpuArray_context(out));
  }
}

int GpuArray_embedding_grad(GpuArray *grad, const GpuArray *dout, const GpuArray *ids, double scale, ssize_t ignore,
                            int accumulate, int check_error) {
  try {
    return embedding_grad(grad, dout, ids, scale, ignore, accumulate, check_error);
  } catch (...) {   // (std::bad_alloc, std::length_error)
    return no_memory(GpuArray_context(grad));
  }
}

int GpuArray_token_logprobs(GpuArray *logp, GpuArray *entropy, GpuArray *stats, GpuArray *top_logp, GpuArray *top_ids,
                            const GpuArray *logits, const GpuArray *ids, double scale, ssize_t ignore,
                            int check_error) {
  try {
    return token_logprobs(logp, entropy, stats, top_logp, top_ids, logits, ids, scale, ignore, check_error);
  } catch (...) {   // (std::bad_alloc, std::length_error)
    return no_memory(GpuArray_context(logits));
  }
}

int GpuArray_token_logprobs_grad(GpuArray *dlogits, const GpuArray *logits, const GpuArray *ids, const GpuArray *stats,
                                 const GpuArray *dlogp, const GpuArray *entropy, const GpuArray *dentropy,
                                 double scale, ssize_t ignore, int check_error) {
  try {
    return token_logprobs_grad(dlogits, logits, ids, stats, dlogp, entropy, dentropy, scale, ignore, check_error);
  } catch (...) {   // (std::bad_alloc, std::length_error)
    return no_memory(GpuArray_context(logits));
  }
}

int GpuGlobalNorm_new(GpuGlobalNorm **g, gpucontext *ctx, const GpuArray **as, GpuArray **rs, size_t n) {
  *g = nullptr;
  try {
    return global_norm_new(g, ctx, as, rs, n);
  } catch (...) {   // (std::bad_alloc, std::length_error)
    return no_memory(ctx);
  }
}

void GpuGlobalNorm_free(GpuGlobalNorm *g) {
  if (g == nullptr) return;
  if (g->table != nullptr) gpudata_release(g->table);
  for (gpudata *b : g->held) gpudata_release(b);
  delete g;
}

int GpuGlobalNorm_norm(const GpuGlobalNorm *g, GpuArray *norm) {
  try {
    return global_norm_call(g, false, 0.0, norm, "GpuGlobalNorm_norm");
  } catch (...) {   // (std::bad_alloc, std::length_error)
    return no_memory(g->ctx);
  }
}

int GpuGlobalNorm_clip(const GpuGlobalNorm *g, double max_norm, GpuArray *norm) {
  try {
    return global_norm_call(g, true, max_norm, norm, "GpuGlobalNorm_clip");
  } catch (...) {   // (std::bad_alloc, std::length_error)
    return no_memory(g->ctx);
  }
}

int GpuArray_global_norm(GpuArray *norm, const GpuArray **as, size_t n) {
  try {
    return norm_and_clip(nullptr, as, n, 0.0, norm, "global_norm");
  } catch (...) {   // (std::bad_alloc, std::length_error)
    return no_memory(GpuArray_context(norm));
  }
}

int GpuArray_clip_global_norm(GpuArray **rs, const GpuArray **as, size_t n, double max_norm, GpuArray *norm) {
  try {
    return norm_and_clip(rs != nullptr ? rs : (GpuArray **)as, as, n, max_norm, norm, "clip_global_norm");
  } catch (...) {   // (std::bad_alloc, std::length_error)
    return n != 0 ? no_memory(GpuArray_context(as[0])) : GA_MEMORY_ERROR;
  }
}

}  // extern "C"
