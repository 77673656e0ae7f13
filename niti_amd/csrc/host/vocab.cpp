// Entries of niti_amd._host for the losses over many classes (see host.h).
#include "host.h"

namespace niti_host {
namespace {

constexpr int64_t kIntMax = 0x7fffffff;

// An int8 tensor [..., features] whose rows are evenly spaced, however far apart: what the kernels read.
struct Rows {
  const int8_t* p;
  int64_t pitch, rows;
};
Rows rows_of(const at::Tensor& t, const char* who, const char* what) {
  if (t.scalar_type() != at::kChar || t.dim() < 1) refuse(std::string(who) + ": " + what + " must be int8 with the features last");
  const int64_t f = t.size(-1);
  int64_t rows = 1, pitch = 0;
  bool even = f <= 1 || t.stride(-1) == 1;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    const int64_t n = t.size(d);
    if (n == 0) return {ptr<int8_t>(t), f, 0};
    if (n == 1) continue;
    if (rows == 1) pitch = t.stride(d);
    else even = even && t.stride(d) == pitch * rows;
    rows *= n;
  }
  if (rows == 1) pitch = f;
  if (!even || pitch < f) refuse(std::string(who) + ": " + what + " must have contiguous features and evenly spaced rows that do not overlap");
  return {ptr<int8_t>(t), pitch, rows};
}

struct Call {
  Rows a, w;
  int rows, features, classes;
};
Call call_of(const at::Tensor& act, const at::Tensor& w, Opt ea, Opt ew, const char* who) {
  if (w.dim() != 2 || act.dim() < 2 || act.size(-1) != w.size(1)) refuse(std::string(who) + ": act [..., features] and w [classes, features] expected");
  if (ea == nullptr || ew == nullptr) refuse(std::string(who) + ": exponents of act and w expected");
  const Call c{rows_of(act, who, "act"), rows_of(w, who, "w"), 0, 0, 0};
  if (w.size(0) < 1 || w.size(1) < 1 || c.a.rows > kIntMax || c.w.rows > kIntMax || w.size(1) > kIntMax)
    refuse(std::string(who) + ": at least one class and one feature, less than 2^31 of each and of the rows");
  return {c.a, c.w, static_cast<int>(c.a.rows), static_cast<int>(w.size(1)), static_cast<int>(c.w.rows)};
}
void same_device(const at::Tensor& like, std::initializer_list<Opt> others, const char* who) {
  for (Opt t : others)
    if (t != nullptr && t->device() != like.device()) refuse(std::string(who) + ": all tensors must live on one GPU");
}
int index_bytes(const at::Tensor& t, const char* who) {
  if (t.scalar_type() == at::kLong) return 8;
  if (t.scalar_type() == at::kInt) return 4;
  refuse(std::string(who) + ": classes must be int64 or int32");
}
// Small ones come out of the stream's own buffer, which stays; large ones go back to the allocator.
at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return bytes <= (32u << 20) ? scratch(bytes, like) : empty8({static_cast<int64_t>(bytes)}, like);
}

// vocab_forward(act, w, exp_a, exp_w, values or None, classes, ignored, temperature) -> (loss, lse, state)
PyObject* forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args g(args, n, 8, "vocab_forward");
    const at::Tensor& act = g.strided();
    const at::Tensor& w = g.strided();
    Opt ea = g.exponent(), ew = g.exponent(), value = g.opt();
    const at::Tensor& index = g.tensor();
    const int64_t ignored = g.integer();
    const double t = g.number();
    const char* const who = value != nullptr ? "vocab_distill" : "vocab_loss";
    const Call c = call_of(act, w, ea, ew, who);
    same_device(act, {&w, ea, ew, value, &index}, who);
    const at::IntArrayRef lead = act.sizes().slice(0, act.dim() - 1);
    const int bytes = index_bytes(index, who);
    int top = 1, type = 0;
    if (value == nullptr) {
      if (index.sizes() != lead) refuse("vocab_loss: one target per row of act expected");
    } else {
      if (index.dim() != act.dim() || index.sizes().slice(0, act.dim() - 1) != lead || value->sizes() != index.sizes() || index.size(-1) < 1)
        refuse("vocab_distill: top_val and top_idx [..., places] with act's rows expected");
      if (index.size(-1) > kIntMax) refuse("vocab_distill: too many places");
      top = static_cast<int>(index.size(-1));
      type = value->scalar_type() == at::kFloat ? NITI_F32 : (value->scalar_type() == at::kBFloat16 ? NITI_BF16 : (value->scalar_type() == at::kHalf ? NITI_F16 : -1));
      if (type < 0) refuse("vocab_distill: top_val must be float32, bfloat16 or float16");
    }
    at::Tensor loss = empty(lead, at::kFloat, act), lse = empty(lead, at::kFloat, act);
    at::Tensor state = empty32({c.rows, static_cast<int64_t>(niti_vocab_state_words(top))}, act);
    if (c.rows > 0) {
      const size_t need = niti_vocab_forward_workspace(c.a.p, c.a.pitch, c.w.p, c.w.pitch, c.rows, c.features, c.classes);
      const at::Tensor ws = workspace(need, act);
      void* const st = stream_of(act);
      if (value == nullptr)
        check(niti_vocab_entropy_i8(c.a.p, c.a.pitch, c.w.p, c.w.pitch, ptr<int32_t>(ea), ptr<int32_t>(ew), c.rows, c.features, c.classes, index.data_ptr(), bytes,
                                    ignored, ptr<float>(loss), ptr<float>(lse), ptr<int32_t>(state), ws.data_ptr(), need, st),
              "niti_vocab_entropy_i8");
      else
        check(niti_vocab_distill_i8(c.a.p, c.a.pitch, c.w.p, c.w.pitch, ptr<int32_t>(ea), ptr<int32_t>(ew), c.rows, c.features, c.classes, value->data_ptr(), type,
                                    index.data_ptr(), bytes, top, static_cast<float>(t), ptr<float>(loss), ptr<float>(lse), ptr<int32_t>(state), ws.data_ptr(), need,
                                    st),
              "niti_vocab_distill_i8");
    }
    return tuple_of({loss, lse, state});
  });
}

// vocab_backward(act, w, exp_a, exp_w, state, places, temperature, weight or None, float32) -> (d_act, d_w)
PyObject* backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args g(args, n, 9, "vocab_backward");
    const at::Tensor& act = g.strided();
    const at::Tensor& w = g.strided();
    Opt ea = g.exponent(), ew = g.exponent();
    const at::Tensor& state = g.tensor();
    const int top = g.i();
    const double t = g.number();
    Opt weight = g.opt();
    const bool f32 = g.flag();
    const char* const who = "vocab_backward";
    const Call c = call_of(act, w, ea, ew, who);
    same_device(act, {&w, ea, ew, &state, weight}, who);
    if (state.scalar_type() != at::kInt || state.dim() != 2 || state.size(0) != c.rows || state.size(1) != static_cast<int64_t>(niti_vocab_state_words(top)))
      refuse("vocab_backward: the state that the forward call of these rows returned expected");
    if (weight != nullptr && (weight->scalar_type() != at::kFloat || (weight->numel() != 1 && weight->sizes() != act.sizes().slice(0, act.dim() - 1))))
      refuse("vocab_backward: grad must be one float32 value or one per row of act");
    const at::ScalarType type = f32 ? at::kFloat : at::kBFloat16;
    at::Tensor da = empty(act.sizes(), type, act), dw = empty(w.sizes(), type, act);
    if (c.rows == 0) {
      dw.zero_();
      return tuple_of({da, dw});
    }
    const auto workspace_of = f32 ? niti_vocab_backward_f32_workspace : niti_vocab_backward_workspace;
    const size_t need = workspace_of(c.a.p, c.a.pitch, c.w.p, c.w.pitch, c.rows, c.features, c.classes);
    const at::Tensor ws = workspace(need, act);
    const int weights = weight == nullptr ? 0 : static_cast<int>(weight->numel());
    if (f32)
      check(niti_vocab_backward_i8_f32(c.a.p, c.a.pitch, c.w.p, c.w.pitch, ptr<int32_t>(ea), ptr<int32_t>(ew), c.rows, c.features, c.classes, top, static_cast<float>(t),
                                       ptr<int32_t>(state), ptr<float>(weight), weights, ptr<float>(da), ptr<float>(dw), ws.data_ptr(), need, stream_of(act)),
            "niti_vocab_backward_i8_f32");
    else
      check(niti_vocab_backward_i8(c.a.p, c.a.pitch, c.w.p, c.w.pitch, ptr<int32_t>(ea), ptr<int32_t>(ew), c.rows, c.features, c.classes, top, static_cast<float>(t),
                                   ptr<int32_t>(state), ptr<float>(weight), weights, ptr<uint16_t>(da), ptr<uint16_t>(dw), ws.data_ptr(), need, stream_of(act)),
            "niti_vocab_backward_i8");
    return tuple_of({da, dw});
  });
}

#define FAST(name) reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr
}  // namespace

PyMethodDef kVocabMethods[] = {{"vocab_forward", FAST(forward)}, {"vocab_backward", FAST(backward)}, {nullptr, nullptr, 0, nullptr}};

}  // namespace niti_host
