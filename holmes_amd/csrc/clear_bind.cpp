// The Python side of the cleartext operators (holmes_amd/clear.py): argument checks, outputs and the C call.
//
// A call on a few tokens costs what the host does for it.  Through ctypes, with the checks in Python, one token's
// attention over two pages took 12.6 us a call, of which the launch is 2.8; from here 6.3 (see clear.py for what
// each function means).  A function returns its tensors, or the C entry point's error code.
#include "clear_args.hpp"

namespace {

Tensor slots_of(PyObject* o, const Pool& p) {
  const Tensor& s = tensor(o, "slots");
  need(s.dim() == 1 && s.scalar_type() == at::kLong && s.device() == p.device,
       "slots must be a 1-d int64 tensor on the pool's device");
  return s.contiguous();
}

// append(pool.., keys, values, slots)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 8);
  const Pool p(a);
  const Tensor &k = tensor(a[5], "keys"), &v = tensor(a[6], "values");
  const Tensor slots = slots_of(a[7], p);
  const int type = type_of(k.scalar_type());
  const int64_t tokens = slots.numel();
  need(type >= 0, "keys must be bfloat16, float16 or float32");
  for (const Tensor* x : {&k, &v})
    if (x->dim() != 3 || x->size(0) != tokens || x->size(1) != p.heads || x->size(2) != p.dim || x->stride(2) != 1 ||
        x->scalar_type() != k.scalar_type() || x->device() != p.device)
      refuse("keys and values must be [" + std::to_string(tokens) + ", " + std::to_string(p.heads) + ", " +
             std::to_string(p.dim) + "], contiguous along the last axis, in one type on the pool's device");
  no_gradient(k, "keys");
  no_gradient(v, "values");
  void* at = p.at();
  const c10::DeviceGuard guard(p.device);
  return PyLong_FromLong(hck_kv4_append(at, p.pages, p.heads, p.dim, type, k.data_ptr(), k.stride(0), k.stride(1),
                                        v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr<int64_t>(), tokens,
                                        stream_of(p.device.index())));
  END_HANDLE_TH_ERRORS
}

// read(pool.., slots, dtype)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 7);
  const Pool p(a);
  const Tensor slots = slots_of(a[5], p);
  if (!THPDtype_Check(a[6])) throw torch::TypeError(std::string("dtype must be a torch.dtype"));
  const ScalarType out = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  const int type = type_of(out);
  need(type >= 0, "dtype must be bfloat16, float16 or float32");
  const int64_t tokens = slots.numel();
  const void* at = p.at();
  const c10::DeviceGuard guard(p.device);
  Tensor k = make({tokens, p.heads, p.dim}, out, p.device), v = make({tokens, p.heads, p.dim}, out, p.device);
  const int err = hck_kv4_read(at, p.pages, p.heads, p.dim, type, slots.data_ptr<int64_t>(), tokens, k.data_ptr(),
                               v.data_ptr(), stream_of(p.device.index()));
  if (err) return PyLong_FromLong(err);
  return Py_BuildValue("(NN)", wrap(std::move(k)), wrap(std::move(v)));
  END_HANDLE_TH_ERRORS
}

// attend(pool.., queries, table, lengths, starts or None, most or None, causal, scale or None, ranges)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 13);
  const Pool p(a);
  const Tensor &q = tensor(a[5], "queries"), &table = tensor(a[6], "table"), &lengths = tensor(a[7], "lengths");
  const int type = type_of(q.scalar_type());
  need(type == HCK_BF16 || type == HCK_F16, "queries must be bfloat16 or float16");
  if (q.dim() != 3 || q.size(2) != p.dim || q.stride(2) != 1 || q.device() != p.device)
    refuse("queries must be [tokens][query heads][" + std::to_string(p.dim) +
           "], contiguous along the last axis, on the pool's device");
  const int64_t tokens = q.size(0), heads = q.size(1);
  if (heads == 0 || heads % p.heads) refuse("query heads must be a multiple of " + std::to_string(p.heads));
  need(table.dim() == 2 && lengths.dim() == 1 && table.size(0) == lengths.size(0),
       "table must be [sequences][columns] and lengths [sequences]");
  const int64_t seqs = table.size(0), cols = table.size(1);
  need(table.scalar_type() == at::kInt && lengths.scalar_type() == at::kInt && table.device() == p.device &&
           lengths.device() == p.device && dense(table, 1) && dense(lengths, 0),
       "table and lengths must be int32 on the pool's device, contiguous along the last axis");
  const int32_t* starts = nullptr;
  if (a[8] != Py_None) {
    const Tensor& s = tensor(a[8], "starts");
    need(s.dim() == 1 && s.size(0) == seqs + 1, "starts must be [sequences + 1], or there is one query for each sequence");
    need(s.scalar_type() == at::kInt && s.device() == p.device && dense(s, 0),
         "starts must be int32 on the pool's device, contiguous along the last axis");
    starts = s.data_ptr<int32_t>();
  } else {
    need(tokens == seqs, "starts must be [sequences + 1], or there is one query for each sequence");
  }
  const int64_t most = a[9] == Py_None ? (starts ? tokens : 1) : std::min<int64_t>(whole(a[9]), tokens);
  need(most >= 0, "most must not be negative");
  const int causal = PyObject_IsTrue(a[10]), ranges = PyObject_IsTrue(a[12]);
  if (causal < 0 || ranges < 0) throw python_error();
  double scale = 1.0 / std::sqrt((double)p.dim);
  if (a[11] != Py_None) {
    scale = PyFloat_AsDouble(a[11]);
    if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  }
  need((float)scale > 0.f && scale <= 0x1p126, "scale must be positive, and 2^126 at most");
  const int64_t group = heads / p.heads;
  // what the C entry point's arguments do not hold, it could not refuse itself
  need(seqs <= INT32_MAX && group <= INT32_MAX && most <= INT32_MAX && cols <= INT32_MAX, "too many sequences, heads or columns");
  no_gradient(q, "queries");
  const void* at = p.at();
  const c10::DeviceGuard guard(p.device);
  Tensor out = make({tokens, heads, p.dim}, q.scalar_type(), p.device), lse = make({tokens, heads}, at::kFloat, p.device);
  Tensor low, high, work;
  if (ranges) {
    low = make({tokens, heads}, at::kFloat, p.device);
    high = make({tokens, heads}, at::kFloat, p.device);
  }
  const size_t bytes =
      hck_kv4_attend_workspace_bytes(tokens, (int)seqs, p.heads, (int)group, p.dim, (int)most, (int)cols);
  if (bytes) work = make({(int64_t)bytes}, at::kByte, p.device);
  const int err = hck_kv4_attend(
      at, p.pages, p.heads, p.dim, type, q.data_ptr(), tokens, (int)group, q.stride(0), q.stride(1),
      table.data_ptr<int32_t>(), table.stride(0), (int)cols, lengths.data_ptr<int32_t>(), starts, (int)seqs, (int)most, causal,
      (float)scale, out.data_ptr(), lse.data_ptr<float>(), ranges ? low.data_ptr<float>() : nullptr,
      ranges ? high.data_ptr<float>() : nullptr, bytes ? work.data_ptr() : nullptr, bytes, stream_of(p.device.index()));
  if (err) return PyLong_FromLong(err);
  return Py_BuildValue("(NNNN)", wrap(std::move(out)), wrap(std::move(lse)), ranges ? wrap(std::move(low)) : none(),
                       ranges ? wrap(std::move(high)) : none());
  END_HANDLE_TH_ERRORS
}

// scores(logits, tokens or None, top)
PyObject* scores(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 3);
  const Tensor& x = tensor(a[0], "logits");
  const int type = type_of(x.scalar_type());
  need(type >= 0, "logits must be bfloat16, float16 or float32");
  need(x.dim() == 2 && x.size(1) >= 1 && dense(x, 1),
       "logits must be [rows][vocabulary], contiguous along the last axis");
  const int64_t rows = x.size(0), vocab = x.size(1);
  const long long top = whole(a[2]), limit = std::min<int64_t>(HCK_TOP_MAX, vocab);
  if (top < 0 || top > limit) refuse("top must be in 0.." + std::to_string(limit));
  need(vocab <= INT32_MAX, "a vocabulary of 2^31 tokens or more");
  Tensor tokens;
  if (a[1] != Py_None) {
    tokens = tensor(a[1], "tokens");
    need(tokens.dim() == 1 && tokens.size(0) == rows && tokens.scalar_type() == at::kLong && tokens.device() == x.device(),
         "tokens must be [rows] int64 on the logits' device");
    tokens = tokens.contiguous();
  }
  if (!x.device().is_cuda()) {
    PyErr_SetString(PyExc_RuntimeError, "token scores run on a GPU: there is no CPU path");
    return nullptr;
  }
  no_gradient(x, "logits");
  const at::Device dev = x.device();
  const c10::DeviceGuard guard(dev);
  Tensor entropy = make({rows}, at::kFloat, dev), given, ids, logs, work;
  if (tokens.defined()) given = make({rows}, at::kFloat, dev);
  if (top) {
    ids = make({rows, top}, at::kLong, dev);
    logs = make({rows, top}, at::kFloat, dev);
  }
  const size_t bytes = hck_token_scores_workspace_bytes(rows, (int)vocab, type, (int)top);
  if (bytes) work = make({(int64_t)bytes}, at::kByte, dev);
  const int err = hck_token_scores(
      x.data_ptr(), type, rows, (int)vocab, x.stride(0), tokens.defined() ? tokens.data_ptr<int64_t>() : nullptr, (int)top,
      tokens.defined() ? given.data_ptr<float>() : nullptr, entropy.data_ptr<float>(), top ? ids.data_ptr<int64_t>() : nullptr,
      top ? logs.data_ptr<float>() : nullptr, bytes ? work.data_ptr() : nullptr, bytes, stream_of(dev.index()));
  if (err) return PyLong_FromLong(err);
  return Py_BuildValue("(NNNN)", tokens.defined() ? wrap(std::move(given)) : none(), wrap(std::move(entropy)),
                       top ? wrap(std::move(ids)) : none(), top ? wrap(std::move(logs)) : none());
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {{"append", (PyCFunction)(void*)append, METH_FASTCALL, nullptr},
                          {"read", (PyCFunction)(void*)read, METH_FASTCALL, nullptr},
                          {"attend", (PyCFunction)(void*)attend, METH_FASTCALL, nullptr},
                          {"scores", (PyCFunction)(void*)scores, METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_clear", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__clear() { return PyModule_Create(&kModule); }
