// The short way from Python into kernels that a step calls with many small tensors: one call takes the tensors themselves, sees that
// they are as the kernel needs them, makes what it returns and launches.  Host code only.  (A call of the smallest sizes, us, from Python tensor
// by tensor with an entry point of plain numbers, and this way: choosing under rules 15.7 and 7.2 to 8.1, adjusting 13.9 and 5.4 to 5.6, attention over
// shared keys 11.7 and 6.1 to 6.4; a launch is 3 of each.)
//
// Every entry point returns a tensor, or None where something is not as it has to be or is none of the usual cases: the caller then goes
// the long way, which says what is wrong.  Loaded with Python's lock held throughout.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include "launch.hpp"

namespace {

// A strided tensor (no subclass of Tensor) on GPU `device`, or null.
const at::Tensor* tensor_on(PyObject* o, int device) {
  if (!o || !THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.layout() == at::kStrided && t.get_device() == device ? &t : nullptr;
}

bool vector_of(PyObject* o, at::ScalarType type, int64_t n, int device, const void*& at) {
  const at::Tensor* t = tensor_on(o, device);
  if (!t || t->scalar_type() != type || t->dim() != 1 || t->size(0) != n || !t->is_contiguous()) return false;
  at = t->data_ptr();
  return true;
}

struct Table { const void* at = nullptr; int64_t ld = 0, rows = 0, columns = 0; };

bool table_of(PyObject* o, int device, Table& x) {
  const at::Tensor* t = tensor_on(o, device);
  if (!t || t->scalar_type() != at::kInt || t->dim() != 2) return false;
  x.rows = t->size(0);
  x.columns = t->size(1);
  x.ld = t->stride(0);
  if ((t->stride(1) != 1 && x.columns > 1) || (x.rows > 1 && x.ld < x.columns)) return false;
  x.ld = x.ld > x.columns ? x.ld : x.columns;
  x.at = t->data_ptr();
  return true;
}

// Attributes of a LogitRules, held while they are in use.
enum { HISTORY, SLOTS, LENGTHS, PROMPT_LENGTHS, REPETITION, PRESENCE, FREQUENCY, BIAS_STARTS, BIAS_TOKENS, BIAS_VALUES, MASKS, MASK_ROWS, ATTRIBUTES };

struct RuleTensors {
  PyObject* o[ATTRIBUTES] = {};
  const void* v[ATTRIBUTES] = {};
  Table history, masks;
  int64_t biases = 0;

  ~RuleTensors() {
    for (PyObject* x : o) Py_XDECREF(x);
  }
  bool read(PyObject* rules, int64_t R, int64_t V, int device) {
    static PyObject* names[ATTRIBUTES];
    if (!names[0]) {
      static const char* const words[ATTRIBUTES] = {"history", "slots", "lengths", "prompt_lengths", "repetition", "presence", "frequency",
                                                    "bias_starts", "bias_tokens", "bias_values", "masks", "mask_rows"};
      for (int i = ATTRIBUTES - 1; i >= 0; --i)
        if (!(names[i] = PyUnicode_InternFromString(words[i]))) return false;
    }
    for (int i = 0; i < ATTRIBUTES; ++i)
      if (!(o[i] = PyObject_GetAttr(rules, names[i]))) return false;
    if (o[HISTORY] != Py_None) {
      if (!table_of(o[HISTORY], device, history)) return false;
      for (int i = SLOTS; i <= PROMPT_LENGTHS; ++i)
        if (!vector_of(o[i], at::kInt, R, device, v[i])) return false;
      for (int i = REPETITION; i <= FREQUENCY; ++i)
        if (!vector_of(o[i], at::kFloat, R, device, v[i])) return false;
    }
    if (o[BIAS_STARTS] != Py_None) {
      const at::Tensor* t = tensor_on(o[BIAS_TOKENS], device);
      if (!t) return false;
      biases = t->numel();
      if (!vector_of(o[BIAS_STARTS], at::kInt, R + 1, device, v[BIAS_STARTS]) || !vector_of(o[BIAS_TOKENS], at::kInt, biases, device, v[BIAS_TOKENS]) ||
          !vector_of(o[BIAS_VALUES], at::kFloat, biases, device, v[BIAS_VALUES]))
        return false;
    }
    if (o[MASKS] != Py_None) {
      if (!table_of(o[MASKS], device, masks) || masks.columns < (V + 31) / 32 || !vector_of(o[MASK_ROWS], at::kInt, R, device, v[MASK_ROWS])) return false;
    }
    const int64_t most = 0x7FFFFFFF;
    return history.rows <= most && history.columns <= most && masks.rows <= most && biases <= most;
  }
};

#define RULE_TYPES                                                                                                                    \
  const void*, long, int, int, const void*, const void*, const void*, const void*, const void*, const void*, const void*, const void*, \
      const void*, int, const void*, long, int, const void*
#define RULE_VALUES(x)                                                                                                               \
  x.history.at, (long)x.history.ld, (int)x.history.rows, (int)x.history.columns, x.v[SLOTS], x.v[LENGTHS], x.v[PROMPT_LENGTHS],       \
      x.v[REPETITION], x.v[PRESENCE], x.v[FREQUENCY], x.v[BIAS_STARTS], x.v[BIAS_TOKENS], x.v[BIAS_VALUES], (int)x.biases, x.masks.at, \
      (long)x.masks.ld, (int)x.masks.rows, x.v[MASK_ROWS]
using Adjust = int (*)(const void*, long, RULE_TYPES, void*, long, int, int, void*);
using Choose = int (*)(const void*, long, RULE_TYPES, const void*, const void*, const void*, void*, void*, void*, int, int, void*);
using Slices = int (*)(int, int);
using Shared = int (*)(const void*, long, const void*, const void*, void*, int, void*, void*, const void*, int, int, const void*, int, const void*, int,
                       int, int, const void*, int, int, int, int, float, float, const void*, void*);

// float32 [rows, vocabulary] with unit inner stride
const at::Tensor* logits_of(PyObject* o, int device) {
  const at::Tensor* t = tensor_on(o, device);
  return t && t->scalar_type() == at::kFloat && t->dim() == 2 && t->stride(1) == 1 && t->size(0) <= 65535 && t->size(1) <= 1 << 30 ? t : nullptr;
}

// Runs f, which returns a new reference or null: None then, and whatever was raised on the way is the long way's to say.
template <typename F>
PyObject* or_none(F f) {
  PyObject* made = nullptr;
  try {
    made = f();
  } catch (...) {
    made = nullptr;
  }
  if (made) return made;
  PyErr_Clear();
  Py_RETURN_NONE;
}

PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

}  // namespace

MIE_EXPORT const char* direct_calls_last_error() { return g_mie_error; }

// adjust: mie_adjust_logits; out: a tensor or None
MIE_EXPORT PyObject* mie_direct_adjust(void* adjust, int device, PyObject* logits, PyObject* rules, PyObject* out, void* stream) {
  return or_none([&]() -> PyObject* {
    const at::Tensor* z = logits_of(logits, device);
    if (!z) return nullptr;
    const int64_t R = z->size(0), V = z->size(1), ld = R > 1 ? z->stride(0) : V;
    RuleTensors x;
    if (!x.read(rules, R, V, device)) return nullptr;
    at::Tensor made;
    const at::Tensor* y;
    if (out == Py_None) {
      made = at::empty({R, V}, z->options());
      y = &made;
    } else {
      y = logits_of(out, device);
      if (!y || y->size(0) != R || y->size(1) != V) return nullptr;
    }
    const int64_t out_ld = R > 1 ? y->stride(0) : V;
    if (out_ld < V) return nullptr;
    const char *a = (const char*)z->data_ptr(), *b = (const char*)y->data_ptr();
    if (a != b || ld != out_ld) {                          // apart from the logits, or the logits themselves
      const int64_t a_bytes = ((R - 1) * ld + V) * 4, b_bytes = ((R - 1) * out_ld + V) * 4;
      if (R > 0 && a < b + b_bytes && b < a + a_bytes) return nullptr;
    }
    if (reinterpret_cast<Adjust>(adjust)(a, ld, RULE_VALUES(x), (void*)b, out_ld, (int)R, (int)V, stream)) return nullptr;
    return out == Py_None ? THPVariable_Wrap(made) : same(out);
  });
}

// choose, slices: mie_choose_by_rules, mie_rules_slices; best, arrived: the stream's workspace, of so many candidates and rows
MIE_EXPORT PyObject* mie_direct_choose(void* choose, void* slices, int device, PyObject* logits, PyObject* rules, PyObject* temperatures, PyObject* seeds,
                                       PyObject* counters, PyObject* out, void* best, void* arrived, long candidates, long rows, void* stream) {
  return or_none([&]() -> PyObject* {
    const at::Tensor* z = logits_of(logits, device);
    if (!z) return nullptr;
    const int64_t R = z->size(0), V = z->size(1);
    const void *t, *s, *c, *chosen;
    if (!vector_of(temperatures, at::kFloat, R, device, t) || !vector_of(seeds, at::kLong, R, device, s) || !vector_of(counters, at::kInt, R, device, c))
      return nullptr;
    RuleTensors x;
    if (!x.read(rules, R, V, device)) return nullptr;
    if (R * reinterpret_cast<Slices>(slices)((int)R, (int)V) > candidates || R > rows) return nullptr;
    at::Tensor made;
    if (out == Py_None) {
      made = at::empty({R}, z->options().dtype(at::kInt));
      chosen = made.data_ptr();
    } else if (!vector_of(out, at::kInt, R, device, chosen)) {
      return nullptr;
    }
    if (reinterpret_cast<Choose>(choose)(z->data_ptr(), R > 1 ? z->stride(0) : V, RULE_VALUES(x), t, s, c, best, arrived, (void*)chosen, (int)R, (int)V, stream))
      return nullptr;
    return out == Py_None ? THPVariable_Wrap(made) : same(out);
  });
}

// What a plan of shared keys says of itself (SharedPrefixPlan.numbers).
struct PlanNumbers {
  long items, row_parts, num_items, whole_items, column_tiles, most_parts, num_parts, rows, q_heads, kv_heads, head_dim, max_context, device;
};

// shared: mie_shared_attention of the plan's head size, for a step that the caller has seen to be the plan's; sinks: float32 [q_heads] or None
MIE_EXPORT PyObject* mie_direct_shared(void* shared, int device, PyObject* qkv, PyObject* k_cache, PyObject* v_cache, PyObject* tables, PyObject* positions,
                                       PyObject* token_row, const PlanNumbers* plan, double scale, double sink_log2,
                                       PyObject* sinks, void* stream) {
  return or_none([&]() -> PyObject* {
    const at::Tensor *q = tensor_on(qkv, device), *k = tensor_on(k_cache, device), *v = tensor_on(v_cache, device), *bt = tensor_on(tables, device);
    if (!q || !k || !v || !bt || q->dim() != 2 || k->dim() != 4 || v->dim() != 4 || bt->dim() != 2) return nullptr;
    const int64_t T = q->size(0), Hq = plan->q_heads, Hkv = plan->kv_heads, D = plan->head_dim, pages = k->size(0), page = k->size(2), blocks = bt->size(1);
    const at::ScalarType type = q->scalar_type();
    if ((type != at::kBFloat16 && type != at::kFloat) || q->stride(1) != 1 || q->size(1) < Hq * D || D % 16 || D < 16 || D > 256) return nullptr;
    if (k->size(1) != Hkv || k->size(3) != D || v->size(0) != pages || v->size(1) != Hkv || v->size(2) != D || v->size(3) != page || page % 16) return nullptr;
    if (k->scalar_type() != type || v->scalar_type() != type || !k->is_contiguous() || !v->is_contiguous()) return nullptr;
    if (bt->scalar_type() != at::kInt || bt->stride(1) != 1 || bt->stride(0) != blocks || bt->size(0) < T) return nullptr;
    if (T != plan->rows || plan->device != device || plan->max_context > blocks * page) return nullptr;
    if (T > 0x7FFFFFFF || pages > 0x7FFFFFFF || blocks > 0x7FFFFFFF || page > 0x7FFFFFFF) return nullptr;
    const void *p, *row, *head_sinks = nullptr;
    if (!vector_of(positions, at::kInt, T, device, p) || !vector_of(token_row, at::kInt, T, device, row)) return nullptr;
    if (sinks != Py_None && !vector_of(sinks, at::kFloat, Hq, device, head_sinks)) return nullptr;
    if (!(scale > 0) || scale > 3e38 || (((uintptr_t)k->data_ptr() | (uintptr_t)v->data_ptr()) & 15)) return nullptr;
    at::Tensor out = at::empty({T, Hq * D}, q->options()), parts;
    float* o_part = nullptr;
    if (plan->most_parts != 1) {                            // partial outputs, then their log-sum-exps
      parts = at::empty({plan->num_parts * Hq * (D + 1)}, q->options().dtype(at::kFloat));
      o_part = (float*)parts.data_ptr();
    }
    if (reinterpret_cast<Shared>(shared)(q->data_ptr(), q->stride(0), k->data_ptr(), v->data_ptr(), out.data_ptr(), type == at::kBFloat16 ? MIE_BF16 : MIE_F32,
                                         o_part, o_part + plan->num_parts * Hq * D, bt->data_ptr(), (int)blocks, (int)pages, p, (int)T, (const void*)plan->items,
                                         (int)plan->num_items, (int)plan->whole_items, (int)plan->column_tiles, (const void*)plan->row_parts,
                                         (int)plan->most_parts, (int)Hq, (int)Hkv, (int)page, (float)(scale * 1.4426950408889634), (float)sink_log2, head_sinks,
                                         stream))
      return nullptr;
    return THPVariable_Wrap(out);
  });
}
