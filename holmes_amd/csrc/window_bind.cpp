// The Python side of the cleartext operators around a prompt and the window of it that is kept (holmes_amd/clear.py):
// rotary positions, attention over whole prompts, the tokens' weights and eviction.  Argument checks, outputs and the C call,
// like clear_bind.cpp.  A function returns its tensors, or the C entry point's error code.
#include "clear_args.hpp"

#include <ATen/ops/clone.h>

namespace {

constexpr int64_t kTokenStride = 1 << 23;  // elements between tokens that hck_prompt_attend takes

int64_t stride_of(const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; }

double scale_of(PyObject* o, int64_t dim) {
  double scale = 1.0 / std::sqrt((double)dim);
  if (o != Py_None) {
    scale = PyFloat_AsDouble(o);
    if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  }
  need((float)scale > 0.f && scale <= 0x1p126, "scale must be positive, and 2^126 at most");
  return scale;
}

bool truth(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw python_error();
  return x;
}

int32_t* ints(const Tensor& t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }

// The starts of `seqs` sequences (fewer than 0: as many as it says), if there are any.
Tensor starts_of(PyObject* o, int64_t seqs, at::Device device) {
  if (o == Py_None) return Tensor();
  const Tensor& s = tensor(o, "starts");
  need(s.dim() == 1 && s.size(0) >= 1 && (seqs < 0 || s.size(0) == seqs + 1), "starts must be [sequences + 1]");
  need(s.scalar_type() == at::kInt && s.device() == device && dense(s, 0),
       "starts must be int32 on the tensors' device, contiguous along the last axis");
  return s;
}

void on_a_gpu(const Tensor& t, const char* what) {
  if (!t.device().is_cuda()) {
    PyErr_SetString(PyExc_RuntimeError, (std::string(what) + " on a GPU: there is no CPU path").c_str());
    throw python_error();
  }
}

// rotate(turns, head_dim, rotated, interleaved, amount, positions, queries, keys or None, inverse)
PyObject* rotate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 9);
  const Tensor &turns = tensor(a[0], "turns"), &q = tensor(a[6], "queries");
  const int64_t dim = whole(a[1]);
  const int rotated = (int)whole(a[2]);
  const bool interleaved = truth(a[3]), inverse = truth(a[8]);
  const double amount = PyFloat_AsDouble(a[4]);
  if (amount == -1.0 && PyErr_Occurred()) throw python_error();
  const at::Device dev = turns.device();
  Tensor positions = tensor(a[5], "positions");
  const int type = type_of(q.scalar_type());
  need(type >= 0, "queries must be bfloat16, float16 or float32");
  const int64_t tokens = q.dim() == 3 ? q.size(0) : 0;
  Tensor k;
  if (a[7] != Py_None) k = tensor(a[7], "keys");
  for (const Tensor* x : {&q, static_cast<const Tensor*>(&k)})
    if (x->defined() && (x->dim() != 3 || x->size(0) != tokens || x->size(2) != dim || !dense(*x, 2) ||
                         x->scalar_type() != q.scalar_type() || x->device() != dev))
      refuse("queries and keys must be [tokens][heads][" + std::to_string(dim) +
             "], contiguous along the last axis, in one type on the plan's device");
  need(positions.dim() == 1 && positions.size(0) == tokens && positions.device() == dev &&
           (positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt),
       "positions must be [tokens] int64 or int32 on the plan's device");
  const int64_t heads = q.size(1), kv_heads = k.defined() ? k.size(1) : 0;
  need(heads + kv_heads <= 65535 && (heads + kv_heads) * dim <= HCK_ROTARY_TOKEN, "too many heads");
  on_a_gpu(turns, "positions are rotated");
  no_gradient(q, "queries");
  if (k.defined()) no_gradient(k, "keys");
  const c10::DeviceGuard guard(dev);
  positions = positions.contiguous();
  Tensor q_out = make({tokens, heads, dim}, q.scalar_type(), dev), k_out;
  if (k.defined()) k_out = make({tokens, kv_heads, dim}, q.scalar_type(), dev);
  const int err = hck_rotary(positions.data_ptr(), positions.scalar_type() == at::kLong ? 8 : 4, tokens,
                             reinterpret_cast<const uint64_t*>(turns.data_ptr<int64_t>()), rotated, interleaved, inverse,
                             (float)amount, type, (int)dim, q.data_ptr(), q.stride(0), q.stride(1), (int)heads,
                             q_out.data_ptr(), k.defined() ? k.data_ptr() : nullptr, k.defined() ? k.stride(0) : 0,
                             k.defined() ? k.stride(1) : 0, (int)kv_heads, k.defined() ? k_out.data_ptr() : nullptr,
                             stream_of(dev.index()));
  if (err) return PyLong_FromLong(err);
  if (!k.defined()) return wrap(std::move(q_out));
  return Py_BuildValue("(NN)", wrap(std::move(q_out)), wrap(std::move(k_out)));
  END_HANDLE_TH_ERRORS
}

// The tensor, or a dense copy of it where its strides or its address are none that 16 bytes can be loaded by.
Tensor loadable(const Tensor& t, bool tokens_apart) {
  bool fine = (uintptr_t)t.data_ptr() % 16 == 0 && stride_of(t, 0) % 8 == 0 && stride_of(t, 1) % 8 == 0;
  if (tokens_apart && t.size(0) > 1) fine = fine && t.stride(0) >= t.size(2) && t.stride(0) <= kTokenStride;
  return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

// prompt(queries, keys, values, starts or None, most or None, causal, scale or None, ranges)
PyObject* prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 8);
  const Tensor &q = tensor(a[0], "queries"), &k = tensor(a[1], "keys"), &v = tensor(a[2], "values");
  const int type = type_of(q.scalar_type());
  need(type == HCK_BF16 || type == HCK_F16, "queries must be bfloat16 or float16");
  const at::Device dev = q.device();
  need(q.dim() == 3 && (q.size(2) == 64 || q.size(2) == 128) && q.stride(2) == 1,
       "queries must be [tokens][query heads][64 or 128], contiguous along the last axis");
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
  for (const Tensor* x : {&k, &v})
    need(x->dim() == 3 && x->size(0) == tokens && x->size(1) == k.size(1) && x->size(2) == dim && x->stride(2) == 1 &&
             x->scalar_type() == q.scalar_type() && x->device() == dev,
         "keys and values must be [tokens][kv_heads][head_dim], contiguous along the last axis, like the queries in type and device");
  const int64_t kv_heads = k.size(1);
  need(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "query heads must be a multiple of the key heads");
  const Tensor starts = starts_of(a[3], -1, dev);
  const int64_t seqs = starts.defined() ? starts.size(0) - 1 : 1;
  const int64_t most = a[4] == Py_None ? tokens : std::min<int64_t>(whole(a[4]), tokens);
  need(most >= 0, "most must not be negative");
  need(tokens <= INT32_MAX && heads <= INT32_MAX && seqs <= INT32_MAX && most * (heads / kv_heads) <= INT32_MAX - 256,
       "too many tokens, heads or sequences");
  const bool causal = truth(a[5]), ranges = truth(a[7]);
  const double scale = scale_of(a[6], dim);
  on_a_gpu(q, "prompts are attended to");
  no_gradient(q, "queries");
  no_gradient(k, "keys");
  no_gradient(v, "values");
  const c10::DeviceGuard guard(dev);
  const Tensor ql = loadable(q, false), kl = loadable(k, true), vl = loadable(v, true);
  Tensor out = make({tokens, heads, dim}, q.scalar_type(), dev), lse = make({tokens, heads}, at::kFloat, dev), low, high;
  if (ranges) {
    low = make({tokens, heads}, at::kFloat, dev);
    high = make({tokens, heads}, at::kFloat, dev);
  }
  const size_t bytes =
      hck_prompt_attend_workspace_bytes(tokens, (int)seqs, (int)kv_heads, (int)(heads / kv_heads), (int)dim, (int)most, causal);
  Tensor work;
  if (bytes) work = make({(int64_t)bytes}, at::kByte, dev);
  const int err = hck_prompt_attend(
      ql.data_ptr(), kl.data_ptr(), vl.data_ptr(), type, tokens, (int)kv_heads, (int)(heads / kv_heads), (int)dim,
      stride_of(ql, 0), stride_of(ql, 1), stride_of(kl, 0), stride_of(kl, 1), stride_of(vl, 0), stride_of(vl, 1), ints(starts),
      (int)seqs, (int)most, causal, scale, out.data_ptr(), lse.data_ptr<float>(), ranges ? low.data_ptr<float>() : nullptr,
      ranges ? high.data_ptr<float>() : nullptr, bytes ? work.data_ptr() : nullptr, bytes, stream_of(dev.index()));
  if (err) return PyLong_FromLong(err);
  return Py_BuildValue("(NNNN)", wrap(std::move(out)), wrap(std::move(lse)), ranges ? wrap(std::move(low)) : none(),
                       ranges ? wrap(std::move(high)) : none());
  END_HANDLE_TH_ERRORS
}

// A table of pages and the sequences' lengths.
void need_table(const Tensor& table, const Tensor& lengths, at::Device device) {
  need(table.dim() == 2 && lengths.dim() == 1 && table.size(0) == lengths.size(0),
       "table must be [sequences][columns] and lengths [sequences]");
  need(table.scalar_type() == at::kInt && lengths.scalar_type() == at::kInt && table.device() == device &&
           lengths.device() == device && dense(table, 1) && dense(lengths, 0),
       "table and lengths must be int32 on the pool's device, contiguous along the last axis");
  need(table.size(0) <= 65535 && table.size(1) < 1 << 23, "more than 65535 sequences, or 2^23 columns");
}

// weigh(pool.., queries, table, lengths, lse, starts or None, most or None, causal, scale or None, prior or None)
PyObject* weigh(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 14);
  const Pool p(a);
  const Tensor &q = tensor(a[5], "queries"), &table = tensor(a[6], "table"), &lengths = tensor(a[7], "lengths");
  const int type = type_of(q.scalar_type());
  need(type == HCK_BF16 || type == HCK_F16, "queries must be bfloat16 or float16");
  if (q.dim() != 3 || q.size(2) != p.dim || q.stride(2) != 1 || q.device() != p.device)
    refuse("queries must be [tokens][query heads][" + std::to_string(p.dim) +
           "], contiguous along the last axis, on the pool's device");
  const int64_t tokens = q.size(0), heads = q.size(1);
  if (heads == 0 || heads % p.heads) refuse("query heads must be a multiple of " + std::to_string(p.heads));
  need_table(table, lengths, p.device);
  const int64_t seqs = table.size(0), cols = table.size(1), group = heads / p.heads;
  Tensor lse = tensor(a[8], "lse");
  need(lse.dim() == 2 && lse.size(0) == tokens && lse.size(1) == heads && lse.scalar_type() == at::kFloat &&
           lse.device() == p.device,
       "lse must be [tokens][query heads] float32 on the pool's device");
  const Tensor starts = starts_of(a[9], seqs, p.device);
  need(starts.defined() || tokens == seqs, "starts must be [sequences + 1], or there is one query for each sequence");
  const int64_t most = a[10] == Py_None ? (starts.defined() ? tokens : 1) : std::min<int64_t>(whole(a[10]), tokens);
  need(most >= 0, "most must not be negative");
  const bool causal = truth(a[11]);
  const double scale = scale_of(a[12], p.dim);
  need(tokens <= INT32_MAX && heads <= INT32_MAX && most * group <= INT32_MAX - 256, "too many tokens or heads");
  Tensor prior;
  if (a[13] != Py_None) {
    prior = tensor(a[13], "prior");
    need(prior.dim() == 3 && prior.size(0) == seqs && prior.size(1) == p.heads && prior.scalar_type() == at::kFloat &&
             prior.device() == p.device && dense(prior, 2) && prior.size(2) <= INT32_MAX,
         "prior must be [sequences][kv_heads][places] float32 on the pool's device, contiguous along the last axis");
    no_gradient(prior, "prior");
  }
  no_gradient(q, "queries");
  no_gradient(lse, "lse");
  const void* at = p.at();
  const c10::DeviceGuard guard(p.device);
  lse = lse.contiguous();
  Tensor out = make({seqs, p.heads, cols * 128}, at::kFloat, p.device);
  const bool has = prior.defined() && prior.numel();
  const size_t bytes = hck_kv4_weigh_workspace_bytes(tokens, (int)seqs, p.heads, (int)group, (int)most, (int)cols);
  Tensor work;
  if (bytes) work = make({(int64_t)bytes}, at::kByte, p.device);
  const int err = hck_kv4_weigh(at, p.pages, p.heads, p.dim, type, q.data_ptr(), tokens, (int)group, q.stride(0), q.stride(1),
                                ints(table), table.stride(0), (int)cols, ints(lengths), ints(starts), (int)seqs, (int)most,
                                causal, scale, lse.data_ptr<float>(), has ? prior.data_ptr<float>() : nullptr,
                                has ? prior.stride(0) : 0, has ? prior.stride(1) : 0, has ? (int)prior.size(2) : 0,
                                out.data_ptr<float>(), bytes ? work.data_ptr() : nullptr, bytes, stream_of(p.device.index()));
  if (err) return PyLong_FromLong(err);
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// evict(pool.., table, lengths, weights, into, keep, recent)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 11);
  const Pool p(a);
  const Tensor &table = tensor(a[5], "table"), &lengths = tensor(a[6], "lengths"), &weights = tensor(a[7], "weights"),
               &into = tensor(a[8], "into");
  need_table(table, lengths, p.device);
  const int64_t seqs = table.size(0);
  need(weights.dim() == 3 && weights.size(0) == seqs && weights.size(1) == p.heads && weights.scalar_type() == at::kFloat &&
           weights.device() == p.device && dense(weights, 2) && weights.size(2) <= INT32_MAX,
       "weights must be [sequences][kv_heads][places] float32 on the pool's device, contiguous along the last axis");
  need(into.dim() == 2 && into.size(0) == seqs && into.scalar_type() == at::kInt && into.device() == p.device &&
           dense(into, 1) && into.size(1) < 1 << 23,
       "into must be [sequences][columns] int32 on the pool's device, contiguous along the last axis");
  const int64_t keep = whole(a[9]), recent = whole(a[10]);
  if (keep < 0 || keep > into.size(1) * 128) refuse("keep must be in 0.." + std::to_string(into.size(1) * 128) + ", what into has room for");
  if (recent < 0 || recent > keep) refuse("recent must be in 0.." + std::to_string(keep));
  no_gradient(weights, "weights");
  void* at = p.at();
  const c10::DeviceGuard guard(p.device);
  Tensor kept = make({seqs, p.heads, keep}, at::kInt, p.device), now = make({seqs}, at::kInt, p.device),
         left = make({seqs, p.heads, keep}, at::kFloat, p.device);
  const size_t bytes = hck_kv4_evict_workspace_bytes((int)seqs, p.heads, (int)table.size(1));
  Tensor work;
  if (bytes) work = make({(int64_t)bytes}, at::kByte, p.device);
  const int err = hck_kv4_evict(at, p.pages, p.heads, p.dim, ints(table), table.stride(0), (int)table.size(1), ints(lengths),
                                (int)seqs, weights.data_ptr<float>(), weights.stride(0), weights.stride(1),
                                (int)weights.size(2), ints(into), into.stride(0), (int)into.size(1), (int)keep, (int)recent,
                                ints(kept), ints(now), left.data_ptr<float>(), bytes ? work.data_ptr() : nullptr, bytes,
                                stream_of(p.device.index()));
  if (err) return PyLong_FromLong(err);
  return Py_BuildValue("(NNN)", wrap(std::move(kept)), wrap(std::move(now)), wrap(std::move(left)));
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {{"rotate", (PyCFunction)(void*)rotate, METH_FASTCALL, nullptr},
                          {"prompt", (PyCFunction)(void*)prompt, METH_FASTCALL, nullptr},
                          {"weigh", (PyCFunction)(void*)weigh, METH_FASTCALL, nullptr},
                          {"evict", (PyCFunction)(void*)evict, METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_window", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__window() { return PyModule_Create(&kModule); }
