// Python calls of the serving operators (module tjkernels._serve): each checks
// its tensors and launches on the current stream of their device.  A step of
// drafted tokens makes two of these calls per layer, on a few tokens: the
// host's share counts (see binding_f8.cpp).

#include "binding.h"

#include <ATen/ops/empty.h>

namespace {

// [tokens, heads, head_dim] with a unit stride of the last dimension.
struct Heads {
  int64_t tokens, heads, hd, ld_token, ld_head;
  int dtype;
  void* data;
};

Heads heads_of(const at::Tensor& t, const char* name) {
  if (t.dim() != 3 || (t.stride(2) != 1 && t.size(2) != 1))
    refuse("%s must be [tokens, heads, head_dim] with a unit stride of the last dimension", name);
  const int64_t ld_head = t.size(1) > 1 ? t.stride(1) : t.size(2);
  return {t.size(0), t.size(1), t.size(2), t.size(0) > 1 ? t.stride(0) : t.size(1) * ld_head, ld_head, dtype_code(t, name),
          t.data_ptr()};
}

// Keys and values [pages, kv_heads, page_size, head_dim], with `layers` in front
// if the caller takes them.
struct Cache {
  tjk_paged_cache c;
  int layers = 1;
  int64_t layer_stride = 0;
};

Cache cache_of(const at::Tensor& k, const at::Tensor& v, bool layered) {
  const int64_t lead = k.dim() - 4;
  if (k.dim() < 4 || lead > (layered ? 1 : 0))
    refuse(layered ? "k_cache must be [pages, kv_heads, page_size, head_dim], with layers in front or not"
                   : "k_cache must be [pages, kv_heads, page_size, head_dim]");
  if (v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type()) refuse("k_cache and v_cache differ in shape or dtype");
  int64_t stride[5];
  for (int64_t d = 0; d < k.dim(); ++d) {
    stride[d] = k.size(d) > 1 ? k.stride(d) : 0;
    if (k.numel() > 0 && stride[d] != (v.size(d) > 1 ? v.stride(d) : 0)) refuse("k_cache and v_cache differ in strides");
  }
  const int64_t *size = k.sizes().data() + lead, *st = stride + lead;
  if (size[3] > 1 && st[3] != 1) refuse("k_cache must have a unit stride of the last dimension");
  for (int64_t d = 1; d < 4; ++d)
    if (size[d] > INT32_MAX) refuse("k_cache is too large");
  Cache r;
  r.c = {k.data_ptr(), v.data_ptr(), st[0], st[1], st[2], size[0], (int)size[2], (int)size[1], (int)size[3],
         dtype_code(k, "k_cache")};
  if (lead) {
    if (k.size(0) > INT32_MAX) refuse("k_cache has too many layers");
    r.layers = (int)k.size(0);
    r.layer_stride = stride[0];
  }
  return r;
}

int32_t* ints(const at::Tensor& t, int64_t n, const char* name) {
  return static_cast<int32_t*>(vector_of(t, n, at::kInt, name));
}

int* errors_of(const at::Tensor* t) {
  if (!t) return nullptr;
  if (t->scalar_type() != at::kInt || t->numel() < 1) refuse("index_errors must be an int32 tensor of at least one element");
  return static_cast<int*>(t->data_ptr());
}

// [batch, columns] of whole numbers with a unit column stride.
struct Table {
  int32_t* data;
  int64_t rows, cols, ld;
};

Table table_of(const at::Tensor& t, const char* name) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || (t.stride(1) != 1 && t.size(1) > 1))
    refuse("%s must be an int32 matrix with a unit column stride", name);
  const int64_t ld = t.size(0) > 1 ? t.stride(0) : t.size(1);
  return {static_cast<int32_t*>(t.data_ptr()), t.size(0), t.size(1), ld};
}

const float* probabilities(const at::Tensor& t, int64_t* rows, int64_t* vocab, int64_t* ld, const char* name) {
  const Matrix m = matrix(t, name);
  if (m.dtype != TJK_F32) refuse("%s must be float32", name);
  *rows = m.rows, *vocab = m.cols, *ld = m.ld;
  return static_cast<const float*>(m.data);
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

// (qkv, positions, table, q_out, k_cache, v_cache, slots, k_out, q_gamma, k_gamma, eps, interleaved, index_errors)
PyObject* rope_append(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded(given, 13, [&] {
    const at::Tensor &qkv_t = tensor(args[0], "qkv"), &pos_t = tensor(args[1], "positions"), &q_t = tensor(args[3], "q_out");
    const at::Tensor *table_t = tensor_or_none(args[2], "table"), *k_t = tensor_or_none(args[4], "k_cache"),
                     *v_t = tensor_or_none(args[5], "v_cache"), *slots_t = tensor_or_none(args[6], "slots"),
                     *ko_t = tensor_or_none(args[7], "k_out"), *qg_t = tensor_or_none(args[8], "q_gamma"),
                     *kg_t = tensor_or_none(args[9], "k_gamma"), *err_t = tensor_or_none(args[12], "index_errors");
    const double eps = real(args[10]);
    const int interleaved = PyObject_IsTrue(args[11]);
    if (interleaved < 0) throw python_error();
    const Heads qkv = heads_of(qkv_t, "qkv"), q = heads_of(q_t, "q_out");
    const int64_t kv2 = qkv.heads - q.heads;
    if (q.heads < 1 || kv2 < 2 || kv2 % 2 || qkv.heads > 1 << 17)
      refuse("qkv has %lld rows a token, q_out %lld: what is left must be keys and values", (long long)qkv.heads,
             (long long)q.heads);
    const int64_t kv = kv2 / 2;
    auto like = [&](const Heads& h, int64_t heads, const char* name) {
      if (h.tokens < qkv.tokens || h.heads != heads || h.hd != qkv.hd || h.dtype != qkv.dtype)
        refuse("%s must be [%lld, %lld, %lld] in qkv's dtype", name, (long long)qkv.tokens, (long long)heads,
               (long long)qkv.hd);
    };
    like(q, q.heads, "q_out");
    Heads ko{};
    if (ko_t) like(ko = heads_of(*ko_t, "k_out"), kv, "k_out");
    if (qkv.hd > INT32_MAX) refuse("head_dim is too large");
    const int32_t* const pos = ints(pos_t, qkv.tokens, "positions");
    int64_t positions = INT32_MAX, rot = 0;
    const float* table = nullptr;
    if (table_t) {
      if (table_t->scalar_type() != at::kFloat || table_t->dim() != 3 || table_t->size(2) != 2 || !table_t->is_contiguous())
        refuse("table must be a contiguous float32 [positions, rotated / 2, 2] tensor");
      positions = table_t->size(0);
      rot = 2 * table_t->size(1);
      table = static_cast<const float*>(table_t->data_ptr());
    }
    Cache cache{};
    const int32_t* slots = nullptr;
    if (!k_t != !v_t || !k_t != !slots_t) refuse("k_cache, v_cache and slots belong together");
    if (k_t) {
      cache = cache_of(*k_t, *v_t, false);
      slots = ints(*slots_t, qkv.tokens, "slots");
    }
    auto gamma = [&](const at::Tensor* t, const char* name) {
      return t ? static_cast<const float*>(vector_of(*t, qkv.hd, at::kFloat, name)) : nullptr;
    };
    const float *qg = gamma(qg_t, "q_gamma"), *kg = gamma(kg_t, "k_gamma");
    int* const err = errors_of(err_t);
    const c10::DeviceIndex device =
        one_device({&qkv_t, &pos_t, table_t, &q_t, k_t, v_t, slots_t, ko_t, qg_t, kg_t, err_t});
    return launch(device, "tjk_rope_append", [&](void* stream) {
      return tjk_rope_append(qkv.data, qkv.ld_token, qkv.ld_head, pos, table, positions, rot, interleaved, q.data, q.ld_token,
                             q.ld_head, ko.data, ko.ld_token, ko.ld_head, k_t ? &cache.c : nullptr, slots, qg, kg, (float)eps,
                             err, qkv.tokens, (int)q.heads, (int)kv, (int)qkv.hd, qkv.dtype, stream);
    });
  });
}

// (q, k_cache, v_cache, block_table, ctx_lens, out, cu_nodes, max_nodes, tree_mask, scale, workspace, index_errors)
PyObject* tree_attention(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded(given, 12, [&] {
    const at::Tensor &q_t = tensor(args[0], "q"), &k_t = tensor(args[1], "k_cache"), &v_t = tensor(args[2], "v_cache"),
                     &bt_t = tensor(args[3], "block_table"), &ctx_t = tensor(args[4], "ctx_lens"),
                     &out_t = tensor(args[5], "out"), &cu_t = tensor(args[6], "cu_nodes"),
                     &ws_t = tensor(args[10], "workspace");
    const at::Tensor *mask_t = tensor_or_none(args[8], "tree_mask"), *err_t = tensor_or_none(args[11], "index_errors");
    const int max_nodes = (int)integer(args[7], "max_nodes");
    const double scale = real(args[9]);
    const Heads q = heads_of(q_t, "q");
    const Cache cache = cache_of(k_t, v_t, false);
    if (q.dtype != cache.c.dtype || q.hd != cache.c.head_dim) refuse("q and the cache differ in dtype or head_dim");
    if (q.heads > 65536) refuse("q has too many heads");
    const Matrix out = matrix(out_t, "out");
    if (out.rows < q.tokens || out.cols != q.heads * q.hd || out.dtype != q.dtype)
      refuse("out must be [%lld, %lld] in q's dtype", (long long)q.tokens, (long long)(q.heads * q.hd));
    const Table bt = table_of(bt_t, "block_table");
    if (bt.rows > INT32_MAX - 1) refuse("block_table has too many rows");
    const int32_t *ctx = ints(ctx_t, bt.rows, "ctx_lens"), *cu = ints(cu_t, bt.rows + 1, "cu_nodes");
    const uint64_t* const mask =
        mask_t ? static_cast<const uint64_t*>(vector_of(*mask_t, q.tokens, at::kLong, "tree_mask")) : nullptr;
    if (!ws_t.is_contiguous()) refuse("workspace must be contiguous");
    int* const err = errors_of(err_t);
    const c10::DeviceIndex device = one_device({&q_t, &k_t, &v_t, &bt_t, &ctx_t, &out_t, &cu_t, mask_t, &ws_t, err_t});
    return launch(device, "tjk_tree_attention", [&](void* stream) {
      return tjk_tree_attention(q.data, q.ld_token, q.ld_head, &cache.c, bt.data, bt.ld, bt.cols, ctx, cu, mask, out.data,
                                out.ld, q.tokens, (int)bt.rows, (int)q.heads, max_nodes, (float)scale, ws_t.data_ptr(),
                                ws_t.nbytes(), err, stream);
    });
  });
}

// (target, draft, tokens, parents, accept_u, sample_u, path, count, token, cu_nodes, workspace, index_errors)
PyObject* verify_tree(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded(given, 12, [&] {
    const at::Tensor &p_t = tensor(args[0], "target"), &q_t = tensor(args[1], "draft"), &tok_t = tensor(args[2], "tokens"),
                     &par_t = tensor(args[3], "parents"), &au_t = tensor(args[4], "accept_u"),
                     &su_t = tensor(args[5], "sample_u"), &path_t = tensor(args[6], "path"),
                     &count_t = tensor(args[7], "count"), &next_t = tensor(args[8], "token"),
                     &cu_t = tensor(args[9], "cu_nodes");
    const at::Tensor *given_t = tensor_or_none(args[10], "workspace"), *err_t = tensor_or_none(args[11], "index_errors");
    int64_t rows, vocab, ld_p, rows_q, vocab_q, ld_q;
    const float* const p = probabilities(p_t, &rows, &vocab, &ld_p, "target");
    const float* const q = probabilities(q_t, &rows_q, &vocab_q, &ld_q, "draft");
    if (rows != rows_q || vocab != vocab_q) refuse("target and draft differ in shape");
    const Table path = table_of(path_t, "path");
    if (path.rows > INT32_MAX - 1 || path.cols > INT32_MAX) refuse("path is too large");
    const int32_t *tok = ints(tok_t, rows, "tokens"), *par = ints(par_t, rows, "parents"),
                  *cu = ints(cu_t, path.rows + 1, "cu_nodes");
    int32_t *count = ints(count_t, path.rows, "count"), *next = ints(next_t, path.rows, "token");
    const float* const au = static_cast<const float*>(vector_of(au_t, rows, at::kFloat, "accept_u"));
    const float* const su = static_cast<const float*>(vector_of(su_t, path.rows, at::kFloat, "sample_u"));
    int* const err = errors_of(err_t);
    if (given_t && !given_t->is_contiguous()) refuse("workspace must be contiguous");
    const c10::DeviceIndex device =
        one_device({&p_t, &q_t, &tok_t, &par_t, &au_t, &su_t, &path_t, &count_t, &next_t, &cu_t, given_t, err_t});
    at::Tensor own;  // freed behind the launch, in the order of the stream
    const size_t need = tjk_verify_tree_bytes(vocab, (int)path.rows);
    if (!given_t && need > 0) own = at::empty({(int64_t)need}, p_t.options().dtype(at::kByte));
    const at::Tensor* const ws_t = given_t ? given_t : need > 0 ? &own : nullptr;
    return launch(device, "tjk_verify_tree", [&](void* stream) {
      return tjk_verify_tree(p, ld_p, q, ld_q, tok, par, au, su, cu, path.data, path.ld, count, next, err, rows, vocab,
                             (int)path.rows, (int)path.cols, ws_t ? ws_t->data_ptr() : nullptr, ws_t ? ws_t->nbytes() : 0,
                             stream);
    });
  });
}

// (k_cache, v_cache, block_table, ctx_lens, path, count, index_errors)
PyObject* compact_cache(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded(given, 7, [&] {
    const at::Tensor &k_t = tensor(args[0], "k_cache"), &v_t = tensor(args[1], "v_cache"),
                     &bt_t = tensor(args[2], "block_table"), &ctx_t = tensor(args[3], "ctx_lens"),
                     &path_t = tensor(args[4], "path"), &count_t = tensor(args[5], "count");
    const at::Tensor* err_t = tensor_or_none(args[6], "index_errors");
    const Cache cache = cache_of(k_t, v_t, true);
    const Table bt = table_of(bt_t, "block_table"), path = table_of(path_t, "path");
    if (bt.rows > INT32_MAX || path.cols > INT32_MAX) refuse("block_table or path is too large");
    if (path.rows != bt.rows) refuse("path must have a row for each of block_table's");
    const int32_t *ctx = ints(ctx_t, bt.rows, "ctx_lens"), *count = ints(count_t, bt.rows, "count");
    int* const err = errors_of(err_t);
    const c10::DeviceIndex device = one_device({&k_t, &v_t, &bt_t, &ctx_t, &path_t, &count_t, err_t});
    return launch(device, "tjk_compact_cache", [&](void* stream) {
      return tjk_compact_cache(&cache.c, cache.layers, cache.layer_stride, bt.data, bt.ld, bt.cols, ctx, path.data, path.ld,
                               (int)path.cols, count, err, (int)bt.rows, stream);
    });
  });
}

PyMethodDef methods[] = {
    {"rope_append", (PyCFunction)(void*)rope_append, METH_FASTCALL, nullptr},
    {"tree_attention", (PyCFunction)(void*)tree_attention, METH_FASTCALL, nullptr},
    {"verify_tree", (PyCFunction)(void*)verify_tree, METH_FASTCALL, nullptr},
    {"compact_cache", (PyCFunction)(void*)compact_cache, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_serve", "Calls of the serving operators.", -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serve(void) { return make_module(&module_def); }
