// exl3_attn.cu -- the C entries of a layer's attention side (include/exl3_b200.h): checks, then the launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <utility>

#include "exl3_attn.h"
#include "exl3_internal.h"

namespace {

constexpr exl3_verdict kOk = {EXL3_OK, nullptr};
exl3_verdict refuse(int32_t code, const char* why) { return {code, why}; }

constexpr int kMaxSeqs = 65535;  // a grid dimension

struct OnDevice {
  int prev = -1;
  explicit OnDevice(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) cudaSetDevice(dev);
    else prev = -1;
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

exl3_verdict launched(cudaError_t e) {
  return e == cudaSuccess ? kOk : refuse(EXL3_FAILED, "exl3_b200: kernel launch failed");
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

exl3_verdict check_cache(const exl3_kv_cache* c) {
  if (!c || c->size != sizeof(exl3_kv_cache) || !c->k || !c->v) return refuse(EXL3_FAILED, "exl3_b200: not a key/value cache");
  if (c->dtype != EXL3_F16 && c->dtype != EXL3_BF16) return refuse(EXL3_UNSUPPORTED, "exl3_b200: the cache holds f16 or bf16");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return refuse(EXL3_UNSUPPORTED, "exl3_b200: head_dim is 64, 128 or 256");
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return refuse(EXL3_UNSUPPORTED, "exl3_b200: page_size is 16, 32, 64, 128 or 256");
  if (c->layers < 1 || c->pages < 1 || c->kv_heads < 1) return refuse(EXL3_FAILED, "exl3_b200: empty cache");
  if (c->kv_heads > 1024 || c->layers > 65536) return refuse(EXL3_TOO_LARGE, "exl3_b200: too many kv heads or layers");
  if (c->pages > (1 << 22)) return refuse(EXL3_TOO_LARGE, "exl3_b200: more than 4194304 pages");
  if (!aligned16(c->k) || !aligned16(c->v) || (c->layer_stride | c->page_stride | c->head_stride | c->token_stride) % 8)
    return refuse(EXL3_UNSUPPORTED, "exl3_b200: cache slots must be 16-byte aligned");
  // nested by stride, every dimension steps over all of the one below it
  std::pair<int64_t, int64_t> dims[4] = {{c->token_stride, c->page_size}, {c->head_stride, c->kv_heads},
                                         {c->page_stride, c->pages}, {c->layer_stride, c->layers}};
  std::sort(dims, dims + 4);
  int64_t span = c->head_dim;
  for (const auto& d : dims) {
    if (d.second == 1) continue;
    if (d.first < span) return refuse(EXL3_FAILED, "exl3_b200: cache slots overlap");
    span += d.first * (d.second - 1);
  }
  return kOk;
}

exl3_verdict check_layer(const exl3_kv_cache* c, int32_t layer) {
  exl3_verdict v = check_cache(c);
  if (v.code != EXL3_OK) return v;
  if (layer < 0 || layer >= c->layers) return refuse(EXL3_FAILED, "exl3_b200: no such layer in the cache");
  return kOk;
}

exl3_verdict check_batch(const exl3_tree_batch* b) {
  if (!b || b->size != sizeof(exl3_tree_batch)) return refuse(EXL3_FAILED, "exl3_b200: not a batch");
  if (b->nseq < 0 || b->rows < 0 || b->max_rows < 0 || b->max_context < 0)
    return refuse(EXL3_FAILED, "exl3_b200: negative batch sizes");
  if (b->nseq > kMaxSeqs) return refuse(EXL3_TOO_LARGE, "exl3_b200: more than 65535 sequences");
  if (b->rows > (1 << 24)) return refuse(EXL3_TOO_LARGE, "exl3_b200: more than 16777216 rows");
  if (b->nseq > 0 && (b->max_pages < 1 || !b->row_start || !b->context || !b->table))
    return refuse(EXL3_FAILED, "exl3_b200: the batch lacks its arrays");
  if (b->tree && b->tree_words < 1) return refuse(EXL3_FAILED, "exl3_b200: a tree without words");
  return kOk;
}

// Heads of a row array; slots of a batch's rows.
exl3_verdict check_heads(const exl3_heads* h, const char* what, int32_t rows, int32_t dim) {
  if (!h || (!h->data && rows > 0)) return refuse(EXL3_FAILED, what);
  if (h->rows != rows || h->dim != dim || h->heads < 1) return refuse(EXL3_FAILED, what);
  return kOk;
}

// Vectors that are written lie apart (those that are only read may repeat: a stride of 0 broadcasts).
bool lies_apart(const exl3_heads* h) {
  const auto step = [](int64_t s) { return s < 0 ? -s : s; };
  const int64_t row = step(h->row_stride), head = step(h->head_stride);
  const bool head_in = h->heads == 1 || head >= h->dim, row_in = h->rows <= 1 || row >= h->dim;
  if (!head_in || !row_in) return false;
  if (h->heads == 1 || h->rows <= 1) return true;
  return row >= head ? row >= head * (h->heads - 1) + h->dim : head >= row * (h->rows - 1) + h->dim;
}

// The bytes of an array of rows of heads: runs of `len` from `base` on, in up to two strides.
struct Runs {
  int64_t base, len;
  int dims = 0;
  int64_t step[2], count[2];
};
Runs runs_of(const exl3_heads* h) {
  const int64_t size = h->dtype == EXL3_F32 ? 4 : 2;
  Runs r{reinterpret_cast<intptr_t>(h->data), h->dim * size};
  std::pair<int64_t, int64_t> d[2] = {{h->head_stride * size, h->heads}, {h->row_stride * size, h->rows}};
  for (auto& [step, count] : d)
    if (step < 0) r.base += step * (count - 1), step = -step;
  if (d[0].first > d[1].first) std::swap(d[0], d[1]);
  for (const auto& [step, count] : d) {
    if (step == 0 || count <= 1) continue;
    if (r.dims == 0 && step == r.len) r.len *= count;  // one run after the other
    else r.step[r.dims] = step, r.count[r.dims++] = count;
  }
  return r;
}
Runs runs_of(const void* p, int64_t bytes) { return {reinterpret_cast<intptr_t>(p), bytes}; }

// Whether some integers k_i in [lo_i, hi_i] bring delta + sum k_i step_i between (below, above): by the longest step first,
// where few k are left.  (Gives up, and says yes, on layouts that need more than `budget` trials.)
struct Term {
  int64_t step, lo, hi;
};
bool hits(const Term* t, int n, int64_t delta, int64_t below, int64_t above, int& budget) {
  if (n == 0) return below < delta && delta < above;
  int64_t least = 0, most = 0;  // what the shorter steps can add
  for (int i = 1; i < n; ++i) least += t[i].lo * t[i].step, most += t[i].hi * t[i].step;
  const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); };
  const int64_t lo = std::max(t->lo, floor_div(below - delta - most, t->step) + 1);
  const int64_t hi = std::min(t->hi, -floor_div(-(above - delta - least), t->step) - 1);
  for (int64_t k = lo; k <= hi; ++k) {
    if (--budget < 0) return true;
    if (hits(t + 1, n - 1, delta + k * t->step, below, above, budget)) return true;
  }
  return false;
}

// Whether two arrays have a byte in common.
bool meet(const Runs& a, const Runs& b) {
  if (a.len <= 0 || b.len <= 0) return false;
  const auto end = [](const Runs& r) {
    int64_t e = r.base + r.len;
    for (int i = 0; i < r.dims; ++i) e += r.step[i] * (r.count[i] - 1);
    return e;
  };
  if (end(a) <= b.base || end(b) <= a.base) return false;
  Term t[4];
  int n = 0;
  for (int i = 0; i < a.dims; ++i) t[n++] = {a.step[i], -(a.count[i] - 1), 0};
  for (int i = 0; i < b.dims; ++i) {
    int j = 0;
    while (j < a.dims && t[j].step != b.step[i]) ++j;
    if (j < a.dims) t[j].hi = b.count[i] - 1;
    else t[n++] = {b.step[i], 0, b.count[i] - 1};
  }
  for (int i = 1; i < n; ++i)
    for (int j = i; j > 0 && t[j].step > t[j - 1].step; --j) std::swap(t[j], t[j - 1]);
  int budget = 4096;
  return hits(t, n, b.base - a.base, -b.len, a.len, budget);
}
bool meet(const exl3_heads* a, const exl3_heads* b) { return meet(runs_of(a), runs_of(b)); }
bool meet(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  return a && b && meet(runs_of(a, a_bytes), runs_of(b, b_bytes));
}
// Whether q_out is q itself: each element is then read by the thread that writes it.
bool same_vectors(const exl3_heads* a, const exl3_heads* b) {
  return a->data == b->data && a->dtype == b->dtype && a->rows == b->rows && a->heads == b->heads &&
         (a->rows <= 1 || a->row_stride == b->row_stride) && (a->heads <= 1 || a->head_stride == b->head_stride);
}

exl3::HeadsView view(const exl3_heads* h) {
  exl3::HeadsView v{};
  v.data = h->data, v.dtype = h->dtype, v.heads = h->heads, v.row_stride = h->row_stride, v.head_stride = h->head_stride;
  const int64_t per = h->dtype == EXL3_F32 ? 4 : 8;  // elements of 16 bytes
  v.vec = aligned16(h->data) && h->row_stride % per == 0 && h->head_stride % per == 0;
  if (v.vec && reinterpret_cast<uintptr_t>(h->data) % 32 == 0 && h->row_stride % (2 * per) == 0 && h->head_stride % (2 * per) == 0)
    v.vec = 2;
  return v;
}

exl3::PagedBatch paged(const exl3_kv_cache* c, int32_t layer, const exl3_tree_batch* b, uint32_t* err) {
  exl3::PagedBatch p{};
  p.k = static_cast<uint16_t*>(c->k) + layer * c->layer_stride;
  p.v = static_cast<uint16_t*>(c->v) + layer * c->layer_stride;
  p.page_stride = c->page_stride, p.head_stride = c->head_stride, p.token_stride = c->token_stride;
  p.pages = c->pages;
  while ((1 << p.page_shift) < c->page_size) ++p.page_shift;
  p.kv_heads = c->kv_heads;
  p.nseq = b->nseq, p.rows = b->rows, p.max_pages = b->max_pages, p.tree_words = b->tree_words;
  p.row_start = b->row_start, p.context = b->context, p.table = b->table, p.tree = b->tree, p.position = b->position;
  p.err = err;
  return p;
}

exl3::PagePool pool_of(const exl3_kv_cache* c) {
  return {static_cast<uint16_t*>(c->k), static_cast<uint16_t*>(c->v), c->layer_stride, c->page_stride, c->head_stride,
          c->token_stride, c->layers, c->kv_heads, c->page_size, c->head_dim};
}

const exl3_verdict kNoWorkspace = {EXL3_FAILED, "exl3_b200: no workspace on this device (exl3_kv_register, exl3_open or a "
                                                "weight load creates it)"};

exl3_verdict check_state(const exl3_page_state* s) {
  if (!s || s->size != sizeof(exl3_page_state) || !s->refs) return refuse(EXL3_FAILED, "exl3_b200: not a page state");
  if (s->nseq < 0 || s->max_pages < 1) return refuse(EXL3_FAILED, "exl3_b200: not a page state");
  if (s->nseq > 0 && (!s->table || !s->held || !s->lens)) return refuse(EXL3_FAILED, "exl3_b200: not a page state");
  if (static_cast<int64_t>(s->nseq) * s->max_pages > (1ll << 30)) return refuse(EXL3_TOO_LARGE, "exl3_b200: page table too large");
  return kOk;
}

// What the page calls share; `moves` in the workspace.  `asked`: the rows' parents or needs.
exl3_verdict page_params(const exl3_kv_cache* cache, const exl3_page_state* in, const exl3_page_state* out,
                         const int32_t* asked, int64_t asked_bytes, const int32_t* missing, exl3::Workspace& ws,
                         exl3::PageParams& p) {
  exl3_verdict v = check_cache(cache);
  if (v.code != EXL3_OK) return v;
  if ((v = check_state(in)).code != EXL3_OK || (v = check_state(out)).code != EXL3_OK) return v;
  if (in->max_pages != out->max_pages) return refuse(EXL3_FAILED, "exl3_b200: the two tables have one width");
  const struct {
    const void* at;
    int64_t bytes;
  } old[4] = {{in->refs, cache->pages * 4ll}, {in->table, in->nseq * 4ll * in->max_pages}, {in->held, in->nseq * 4ll},
              {in->lens, in->nseq * 4ll}},
    made[5] = {{out->refs, cache->pages * 4ll}, {out->table, out->nseq * 4ll * out->max_pages}, {out->held, out->nseq * 4ll},
               {out->lens, out->nseq * 4ll}, {missing, 4}};
  for (const auto& m : made) {
    for (const auto& o : old)
      if (meet(m.at, m.bytes, o.at, o.bytes)) return refuse(EXL3_FAILED, "exl3_b200: the new page state has its own arrays");
    if (meet(m.at, m.bytes, asked, asked_bytes))
      return refuse(EXL3_FAILED, "exl3_b200: the new page state lies over the call's arguments");
  }
  for (int i = 0; i < 4; ++i)
    if (meet(missing, 4, made[i].at, made[i].bytes))
      return refuse(EXL3_FAILED, "exl3_b200: the new page state lies over the call's arguments");
  if (!exl3::workspace_get(cache->device, ws)) return kNoWorkspace;
  p = {};
  p.pages = cache->pages;
  while ((1 << p.page_shift) < cache->page_size) ++p.page_shift;
  p.nseq_in = in->nseq, p.nseq_out = out->nseq, p.width_in = in->max_pages, p.width_out = out->max_pages;
  p.refs_in = in->refs, p.table_in = in->table, p.held_in = in->held, p.lens_in = in->lens;
  p.refs = out->refs, p.table = out->table, p.held = out->held, p.lens = out->lens;
  p.moves = reinterpret_cast<int32_t*>(ws.partials);
  p.err = ws.err;
  return kOk;
}

}  // namespace

extern "C" {

exl3_verdict exl3_kv_register(const exl3_kv_cache* cache) {
  exl3_verdict v = check_cache(cache);
  return v.code == EXL3_OK ? exl3::workspace_create(cache->device) : v;
}

exl3_verdict exl3_qk_norm_rope(const exl3_kv_cache* cache, int32_t layer, const exl3_tree_batch* batch,
                               const exl3_heads* q, const exl3_heads* k, const exl3_heads* v,
                               const exl3_norm_rope* opts, void* stream, const exl3_heads* q_out) {
  exl3_verdict r = check_layer(cache, layer);
  if (r.code != EXL3_OK || (r = check_batch(batch)).code != EXL3_OK) return r;
  const int32_t rows = batch->rows, dim = cache->head_dim;
  if ((r = check_heads(q, "exl3_b200: q is [rows, heads, head_dim]", rows, dim)).code != EXL3_OK) return r;
  if ((r = check_heads(k, "exl3_b200: k is [rows, kv_heads, head_dim]", rows, dim)).code != EXL3_OK) return r;
  if ((r = check_heads(v, "exl3_b200: v is [rows, kv_heads, head_dim]", rows, dim)).code != EXL3_OK) return r;
  if ((r = check_heads(q_out, "exl3_b200: q_out is [rows, heads, head_dim]", rows, dim)).code != EXL3_OK) return r;
  if (k->heads != cache->kv_heads || v->heads != cache->kv_heads)
    return refuse(EXL3_FAILED, "exl3_b200: k and v have the cache's kv heads");
  if (q_out->heads != q->heads) return refuse(EXL3_FAILED, "exl3_b200: q_out has q's heads");
  if (q->dtype != EXL3_F16 && q->dtype != EXL3_BF16 && q->dtype != EXL3_F32)
    return refuse(EXL3_UNSUPPORTED, "exl3_b200: q, k and v are f16, bf16 or f32");
  if (k->dtype != q->dtype || v->dtype != q->dtype) return refuse(EXL3_UNSUPPORTED, "exl3_b200: q, k and v have one dtype");
  if (q_out->dtype != q->dtype && q_out->dtype != cache->dtype)
    return refuse(EXL3_UNSUPPORTED, "exl3_b200: q_out has q's dtype or the cache's");
  if (!lies_apart(q_out)) return refuse(EXL3_FAILED, "exl3_b200: q_out's vectors overlap");
  if (q_out->data && meet(q_out, q) && !same_vectors(q_out, q))
    return refuse(EXL3_FAILED, "exl3_b200: q_out lies over q in another layout");
  if (!opts || opts->size != sizeof(exl3_norm_rope)) return refuse(EXL3_FAILED, "exl3_b200: not norm and rotation options");
  if (opts->rot_dims < 0 || opts->rot_dims > dim || opts->rot_dims % 2 || (!opts->adjacent && opts->rot_dims % 16))
    return refuse(EXL3_UNSUPPORTED, "exl3_b200: rot_dims is even, at most head_dim, and a multiple of 16 for split halves");
  if (opts->rot_dims && !opts->inv_freq) return refuse(EXL3_FAILED, "exl3_b200: rotation without frequencies");
  if ((opts->q_weight || opts->k_weight) && opts->weight_dtype != EXL3_F16 && opts->weight_dtype != EXL3_BF16 &&
      opts->weight_dtype != EXL3_F32)
    return refuse(EXL3_UNSUPPORTED, "exl3_b200: norm weights are f16, bf16 or f32");
  if (!(opts->eps >= 0.f)) return refuse(EXL3_FAILED, "exl3_b200: eps is not negative");
  if (batch->nseq == 0 || rows == 0) return kOk;
  if (meet(q_out, k) || meet(q_out, v)) return refuse(EXL3_FAILED, "exl3_b200: q_out lies over k or v");
  exl3::Workspace ws;
  if (!exl3::workspace_get(cache->device, ws)) return kNoWorkspace;
  OnDevice guard(cache->device);
  exl3::NormRopeParams p{};
  p.b = paged(cache, layer, batch, ws.err);
  p.q = view(q), p.k = view(k), p.v = view(v), p.out = view(q_out);
  p.q_weight = opts->q_weight, p.k_weight = opts->k_weight, p.inv_freq = opts->inv_freq;
  p.dim = dim, p.rot_dims = opts->rot_dims, p.adjacent = opts->adjacent, p.weight_dtype = opts->weight_dtype;
  p.cache_dtype = cache->dtype;
  p.eps = opts->eps, p.weight_offset = opts->weight_offset;
  return launched(exl3::launch_norm_rope(p, ws.sms, static_cast<cudaStream_t>(stream)));
}

exl3_verdict exl3_tree_attention(const exl3_kv_cache* cache, int32_t layer, const exl3_tree_batch* batch,
                                 const exl3_heads* q, float scale, void* stream, const exl3_heads* out, float* lse) {
  exl3_verdict r = check_layer(cache, layer);
  if (r.code != EXL3_OK || (r = check_batch(batch)).code != EXL3_OK) return r;
  const int32_t rows = batch->rows, dim = cache->head_dim;
  if ((r = check_heads(q, "exl3_b200: q is [rows, heads, head_dim]", rows, dim)).code != EXL3_OK) return r;
  if ((r = check_heads(out, "exl3_b200: out is [rows, heads, head_dim]", rows, dim)).code != EXL3_OK) return r;
  if (q->dtype != cache->dtype || out->dtype != cache->dtype)
    return refuse(EXL3_UNSUPPORTED, "exl3_b200: q and out have the cache's dtype");
  if (out->heads != q->heads || q->heads % cache->kv_heads)
    return refuse(EXL3_FAILED, "exl3_b200: q and out have a whole number of heads per kv head");
  if (!lies_apart(out)) return refuse(EXL3_FAILED, "exl3_b200: out's vectors overlap");
  if (q->heads > 4096) return refuse(EXL3_TOO_LARGE, "exl3_b200: more than 4096 query heads");
  if (static_cast<int64_t>(rows) * q->heads > (1ll << 30)) return refuse(EXL3_TOO_LARGE, "exl3_b200: more than 2^30 query vectors");
  if (!(scale > 0.f) || std::isinf(scale)) return refuse(EXL3_UNSUPPORTED, "exl3_b200: the scale is a positive number");
  if (batch->max_rows > rows) return refuse(EXL3_FAILED, "exl3_b200: max_rows is above the batch's rows");
  if (batch->nseq == 0 || rows == 0) return kOk;
  if (meet(out, q)) return refuse(EXL3_FAILED, "exl3_b200: out is not q (a row may be read again at its end)");
  if (lse) {
    const Runs l = runs_of(lse, static_cast<int64_t>(rows) * q->heads * 4);
    if (meet(l, runs_of(q)) || meet(l, runs_of(out))) return refuse(EXL3_FAILED, "exl3_b200: lse lies over q or out");
  }
  exl3::Workspace ws;
  if (!exl3::workspace_get(cache->device, ws)) return kNoWorkspace;
  OnDevice guard(cache->device);
  exl3::AttnParams p{};
  p.b = paged(cache, layer, batch, ws.err);
  p.q = view(q), p.out = view(out);
  p.lse = lse;
  p.group = q->heads / cache->kv_heads;
  p.bf16 = cache->dtype == EXL3_BF16;
  p.max_rows = batch->max_rows > 0 ? batch->max_rows : rows;
  const int64_t width = static_cast<int64_t>(batch->max_pages) * cache->page_size;
  if (width > 0x7FFF0000) return refuse(EXL3_TOO_LARGE, "exl3_b200: the table spans 2^31 slots or more");
  p.max_context = static_cast<int32_t>(batch->max_context > 0 && batch->max_context < width ? batch->max_context : width);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.partials = ws.partials, p.counters = ws.counters;
  const bool few = static_cast<int64_t>(p.max_rows) * p.group <= exl3::attn_few_rows(dim);
  return launched((few ? exl3::launch_attn_mma : exl3::launch_attn_tc)(p, dim, ws.sms, ws.partial_floats,
                                                                       static_cast<cudaStream_t>(stream)));
}

exl3_verdict exl3_cache_fork(const exl3_kv_cache* cache, const exl3_page_state* in, const int32_t* parent, void* stream,
                             const exl3_page_state* out) {
  // every old row looks through the new rows for its children
  if (in && out && in->nseq > 0 && out->nseq > 0 && static_cast<int64_t>(in->nseq) * out->nseq > (1ll << 32))
    return refuse(EXL3_TOO_LARGE, "exl3_b200: fork takes at most 2^32 pairs of an old and a new row");
  exl3::Workspace ws;
  exl3::PageParams p;
  exl3_verdict v = page_params(cache, in, out, parent, out ? out->nseq * 4ll : 0, nullptr, ws, p);
  if (v.code != EXL3_OK) return v;
  if (!parent && out->nseq > 0) return refuse(EXL3_FAILED, "exl3_b200: fork without parents");
  p.parent = parent;
  OnDevice guard(cache->device);
  return launched(exl3::launch_cache_fork(p, static_cast<cudaStream_t>(stream)));
}

exl3_verdict exl3_cache_grow(const exl3_kv_cache* cache, const exl3_page_state* in, const int32_t* need, void* stream,
                             const exl3_page_state* out, int32_t* missing) {
  exl3::Workspace ws;
  exl3::PageParams p;
  exl3_verdict v = page_params(cache, in, out, need, in ? in->nseq * 4ll : 0, missing, ws, p);
  if (v.code != EXL3_OK) return v;
  if (in->nseq != out->nseq) return refuse(EXL3_FAILED, "exl3_b200: grow keeps the rows");
  if (in->nseq > exl3::cache_grow_max_rows()) return refuse(EXL3_TOO_LARGE, "exl3_b200: grow takes at most 4096 rows");
  if (!missing || (!need && in->nseq > 0)) return refuse(EXL3_FAILED, "exl3_b200: grow without its arrays");
  if (ws.partial_floats < static_cast<size_t>(in->nseq) * 5 + static_cast<size_t>(cache->pages) * 2 + 1)
    return refuse(EXL3_TOO_LARGE, "exl3_b200: too many pages for the workspace");
  p.need = need, p.missing = missing;
  p.scratch = p.moves + 1 + 2 * in->nseq;
  OnDevice guard(cache->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  v = launched(exl3::launch_cache_grow(p, st));
  if (v.code != EXL3_OK) return v;
  return launched(exl3::launch_page_copy(pool_of(cache), p.moves, in->nseq, ws.sms, st));
}

exl3_verdict exl3_cache_compact(const exl3_kv_cache* cache, const exl3_page_state* in, void* stream,
                                const exl3_page_state* out) {
  exl3::Workspace ws;
  exl3::PageParams p;
  exl3_verdict v = page_params(cache, in, out, nullptr, 0, nullptr, ws, p);
  if (v.code != EXL3_OK) return v;
  if (in->nseq != out->nseq) return refuse(EXL3_FAILED, "exl3_b200: compact keeps the rows");
  if (ws.partial_floats < static_cast<size_t>(cache->pages) * 4 + 1)
    return refuse(EXL3_TOO_LARGE, "exl3_b200: too many pages for the workspace");
  OnDevice guard(cache->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  v = launched(exl3::launch_cache_compact(p, st));
  if (v.code != EXL3_OK) return v;
  return launched(exl3::launch_page_copy(pool_of(cache), p.moves, cache->pages / 2 + 1, ws.sms, st));
}

exl3_verdict exl3_cache_keep(const exl3_kv_cache* cache, const exl3_tree_batch* batch, const int32_t* path,
                             int32_t depth, const int32_t* kept, void* stream, int32_t* lens) {
  exl3_verdict r = check_cache(cache);
  if (r.code != EXL3_OK || (r = check_batch(batch)).code != EXL3_OK) return r;
  if (batch->nseq == 0) return kOk;
  if (!kept || !lens) return refuse(EXL3_FAILED, "exl3_b200: keep without its arrays");
  if (path && depth < 1) return refuse(EXL3_FAILED, "exl3_b200: a path without depth");
  const int64_t bytes = batch->nseq * 4ll;
  if ((lens != batch->context && meet(lens, bytes, batch->context, bytes)) || (lens != kept && meet(lens, bytes, kept, bytes)) ||
      meet(lens, bytes, path, bytes * depth) || meet(lens, bytes, batch->table, bytes * batch->max_pages) ||
      meet(lens, bytes, batch->row_start, bytes + 4))
    return refuse(EXL3_FAILED, "exl3_b200: lens lies over the call's arguments");
  exl3::Workspace ws;
  if (!exl3::workspace_get(cache->device, ws)) return kNoWorkspace;
  OnDevice guard(cache->device);
  exl3::KeepParams p{};
  p.pool = pool_of(cache);
  p.b = paged(cache, 0, batch, ws.err);
  p.path = path, p.depth = depth, p.kept = kept, p.lens = lens;
  if (lens == batch->context || lens == kept) p.counters = ws.counters;
  return launched(exl3::launch_cache_keep(p, ws.counter_count, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
