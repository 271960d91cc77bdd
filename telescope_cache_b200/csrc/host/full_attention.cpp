// Host side of the full-attention operators (rotary positions, packed causal
// attention, 8-bit cache): argument checks, outputs and workspaces, and the call
// of the library's C entry, without the interpreter in between.  A ctypes call
// that fills these argument blocks field by field costs 20 to 40 us, several
// times the kernels of a decode step.
//
// Every function raises ValueError on arguments that do not go together,
// RuntimeError on tensors that are not on a CUDA device (there is no CPU path),
// TypeError on other element types.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <map>
#include <stdexcept>
#include <string>
#include <tuple>

#include "../../../include/telescope_cache.h"

namespace py = pybind11;

// Python exceptions with the message alone.
#define CHECK_VALUE(cond, ...) \
  do {                         \
    if (!(cond)) throw py::value_error(c10::str(__VA_ARGS__)); \
  } while (0)
#define CHECK_RUN(cond, ...) \
  do {                       \
    if (!(cond)) throw std::runtime_error(c10::str(__VA_ARGS__)); \
  } while (0)

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

int dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return TC_F32;
  if (t == at::kBFloat16) return TC_BF16;
  if (t == at::kHalf) return TC_F16;
  throw py::type_error(c10::str("telescope_cache_b200: unsupported dtype ", t));
}

void cuda(const Tensor& t) {
  CHECK_RUN(t.is_cuda(), "telescope_cache_b200 computes on CUDA tensors only (got a tensor on ", t.device(),
              "); there is no CPU fallback");
}
void same_device(const Tensor& a, const Tensor& b) {
  cuda(b);
  CHECK_VALUE(a.device() == b.device(), "tensors on ", a.device(), " and ", b.device());
}

[[noreturn]] void not_implemented(const std::string& what) {
  PyErr_SetString(PyExc_NotImplementedError, what.c_str());
  throw py::error_already_set();
}
void done(int rc, const char* what) {
  if (rc == TC_OK) return;
  const std::string text = c10::str("telescope_cache_b200: ", what, " failed with status ", rc);
  if (rc == TC_ERR_ARG || rc == TC_ERR_SCHEDULE) CHECK_VALUE(false, text);
  if (rc == TC_ERR_UNSUPPORTED) not_implemented(text);
  CHECK_RUN(false, text);
}

// A tangent would be dropped without a word.
void no_tangent(const Tensor& t) {
  if (t._fw_grad(0).defined()) not_implemented("telescope_cache_b200: forward-mode derivatives are not supported");
}

// The factor of q.k, 1 / sqrt(D) unless given.
float scale_of(std::optional<double> scale, int64_t D) {
  CHECK_VALUE(!scale || std::isfinite((float)*scale), "scale must be finite, got ", scale.value_or(0.));
  return (float)scale.value_or(1.0 / std::sqrt((double)D));
}

void check_softcap(std::optional<double> softcap) {
  CHECK_VALUE(!softcap || ((float)*softcap > 0.f && std::isfinite((float)*softcap)), "softcap must be positive and finite, got ",
              softcap.value_or(0.));
}

int32_t i32(int64_t v, const char* what) {
  CHECK_VALUE(v >= 0 && v <= INT32_MAX, what, " of ", v, " does not fit 31 bits");
  return (int32_t)v;
}

Tensor dense_head(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
Tensor table(const Tensor& t) {
  return t.scalar_type() == at::kFloat && t.is_contiguous() ? t : t.to(at::kFloat).contiguous();
}
bool integral(const Tensor& t) {
  const auto k = t.scalar_type();
  return k == at::kInt || k == at::kLong || k == at::kShort || k == at::kChar || k == at::kByte;
}
// Indices (positions, cache rows) as int32: one of 64 bits that does not fit goes to
// the nearest that is no index.
Tensor indices(const Tensor& t) {
  return (t.scalar_type() == at::kLong ? t.clamp(-1, INT32_MAX) : t).to(at::kInt).contiguous();
}

// The device status word: one int32 per device, shared with the Python layer.
std::map<int, Tensor>& status_words() {
  static auto* m = new std::map<int, Tensor>;
  return *m;
}
int32_t* status_of(const Tensor& t) {
  auto it = status_words().find(t.device().index());
  return it == status_words().end() ? nullptr : it->second.data_ptr<int32_t>();
}
void set_status(const Tensor& word) { status_words()[word.device().index()] = word; }

struct Call {  // device and stream of a call
  c10::cuda::CUDAGuard guard;
  cudaStream_t stream;
  explicit Call(const Tensor& t) : guard(t.device()), stream(at::cuda::getCurrentCUDAStream(t.device().index())) {}
};

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
std::tuple<Tensor, OptTensor> rotary(const Tensor& q0, const OptTensor& k0, const Tensor& cos0, const Tensor& sin0,
                                     const OptTensor& positions, bool interleaved, bool inverse) {
  CHECK_VALUE(q0.dim() == 4, "q must be [B, N, H, D], got ", q0.sizes());
  const int64_t B = q0.size(0), N = q0.size(1), D = q0.size(3);
  if (k0) {
    CHECK_VALUE(k0->dim() == 4 && k0->size(0) == B && k0->size(1) == N && k0->size(3) == D, "k shape ", k0->sizes(),
                      " incompatible with q ", q0.sizes());
    CHECK_VALUE(k0->scalar_type() == q0.scalar_type(), "k dtype ", k0->scalar_type(), " must match q dtype ",
                      q0.scalar_type());
  }
  CHECK_VALUE(cos0.dim() == 2 && cos0.sizes() == sin0.sizes(), "cos ", cos0.sizes(), " and sin ", sin0.sizes(),
                    " must be one [n_pos, R / 2] shape");
  CHECK_VALUE(2 * cos0.size(1) <= D, "rotary tables cover dim ", 2 * cos0.size(1), ", the heads have ", D);
  cuda(q0);
  if (k0) same_device(q0, *k0);
  same_device(q0, cos0);
  same_device(q0, sin0);
  for (const Tensor* t : {&q0, &cos0, &sin0}) no_tangent(*t);
  if (k0) no_tangent(*k0);
  Tensor pos;
  if (positions) {
    const bool shared = positions->dim() == 1 && positions->size(0) == N;
    CHECK_VALUE(integral(*positions) && (shared || (positions->dim() == 2 && positions->size(0) == B && positions->size(1) == N)),
                      "positions must be integers [", N, "] or [", B, ", ", N, "], got ", positions->sizes(), " ",
                      positions->scalar_type());
    same_device(q0, *positions);
    pos = indices(*positions);
  } else {
    CHECK_VALUE(cos0.size(0) >= N, "rotary tables cover ", cos0.size(0), " positions, q has ", N);
  }
  Call call(q0);
  const Tensor q = dense_head(q0), cos = table(cos0), sin = table(sin0);
  tc_rotary_args a{};
  a.B = i32(B, "batch"), a.N = i32(N, "length"), a.Hq = i32(q.size(2), "heads"), a.D = i32(D, "head dim");
  a.R = (int32_t)(2 * cos.size(1)), a.dtype = dtype_code(q.scalar_type());
  a.interleaved = interleaved, a.inverse = inverse, a.n_pos = i32(cos.size(0), "table length");
  Tensor qo = at::empty(q.sizes(), q.options());
  a.q = q.data_ptr(), a.q_stride_b = q.stride(0), a.q_stride_n = q.stride(1), a.q_stride_h = q.stride(2), a.q_out = qo.data_ptr();
  Tensor k, ko;
  if (k0) {
    k = dense_head(*k0);
    ko = at::empty(k.sizes(), k.options());
    a.Hk = i32(k.size(2), "heads");
    a.k = k.data_ptr(), a.k_stride_b = k.stride(0), a.k_stride_n = k.stride(1), a.k_stride_h = k.stride(2), a.k_out = ko.data_ptr();
  }
  a.cos_t = cos.data_ptr<float>(), a.sin_t = sin.data_ptr<float>();
  if (pos.defined()) a.positions = pos.data_ptr<int32_t>(), a.pos_stride_b = pos.dim() == 2 ? N : 0;
  done(tc_rotary(&a, call.stream), "tc_rotary");
  return {qo, k0 ? OptTensor(ko) : std::nullopt};
}

// ---------------------------------------------------------------------------
// packed causal attention
// ---------------------------------------------------------------------------
std::tuple<Tensor, Tensor> segment_bounds(const Tensor& seq_idx) {
  CHECK_VALUE(seq_idx.dim() == 2 && integral(seq_idx), "seq_idx must be an integer tensor [B, N], got ",
                    seq_idx.sizes(), " ", seq_idx.scalar_type());
  cuda(seq_idx);
  Call call(seq_idx);
  const bool wide = seq_idx.scalar_type() == at::kLong;  // ids of 64 bits are compared as they are
  const Tensor ids = (wide ? seq_idx : seq_idx.to(at::kInt)).contiguous();
  Tensor both = at::empty({2, ids.size(0), ids.size(1)}, ids.options().dtype(at::kInt));
  Tensor starts = both.select(0, 0), ends = both.select(0, 1);
  const int32_t B = i32(ids.size(0), "batch"), N = i32(ids.size(1), "length");
  int32_t *s = starts.data_ptr<int32_t>(), *e = ends.data_ptr<int32_t>();
  done(wide ? tc_segment_bounds_i64(B, N, ids.data_ptr<int64_t>(), s, e, call.stream)
            : tc_segment_bounds(B, N, ids.data_ptr<int32_t>(), s, e, call.stream),
       "tc_segment_bounds");
  return {starts, ends};
}

struct Causal {
  Tensor q, k, v, starts, ends;
  tc_causal_args a{};
};

// seq: example ids [B, N]; or starts and ends, the bounds already formed.
void causal_args(Causal& c, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& seq, const OptTensor& starts,
                 const OptTensor& ends, std::optional<double> softcap, std::optional<double> scale, int impl) {
  CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k, v must be [B, N, H, D], got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  const int64_t B = q.size(0), N = q.size(1), Hq = q.size(2), Dk = q.size(3), Hkv = k.size(2);
  CHECK_VALUE(k.size(0) == B && k.size(1) == N && k.size(3) == Dk, "k shape ", k.sizes(), " incompatible with q ", q.sizes());
  CHECK_VALUE(v.size(0) == B && v.size(1) == N && v.size(2) == Hkv, "v shape ", v.sizes(), " incompatible with k ", k.sizes());
  CHECK_VALUE(Hkv != 0 && Hq % Hkv == 0, "Hq=", Hq, " must be divisible by Hkv=", Hkv, ".");
  CHECK_VALUE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
                    "q, k, v must share a dtype, got ", q.scalar_type(), ", ", k.scalar_type(), ", ", v.scalar_type());
  check_softcap(softcap);
  CHECK_VALUE(starts.has_value() == ends.has_value(), "segment starts and ends go together");
  cuda(q);
  same_device(q, k);
  same_device(q, v);
  if (seq) {
    CHECK_VALUE(seq->dim() == 2 && seq->size(0) == B && seq->size(1) == N && integral(*seq),
                      "seq_idx must be an integer tensor [", B, ", ", N, "], got ", seq->sizes(), " ", seq->scalar_type());
    same_device(q, *seq);
    std::tie(c.starts, c.ends) = segment_bounds(*seq);
  } else if (starts) {
    for (const Tensor* t : {&*starts, &*ends}) {
      CHECK_VALUE(t->dim() == 2 && t->size(0) == B && t->size(1) == N && t->scalar_type() == at::kInt,
                        "segment bounds ", t->sizes(), " != [", B, ", ", N, "] int32");
      same_device(q, *t);
    }
    c.starts = starts->contiguous(), c.ends = ends->contiguous();
  }
  c.q = dense_head(q), c.k = dense_head(k), c.v = dense_head(v);
  tc_causal_args& a = c.a;
  a.B = i32(B, "batch"), a.N = i32(N, "length"), a.Hq = i32(Hq, "heads"), a.Hkv = i32(Hkv, "heads");
  a.Dk = i32(Dk, "head dim"), a.Dv = i32(v.size(3), "head dim"), a.dtype = dtype_code(q.scalar_type());
  a.has_softcap = softcap.has_value(), a.softcap = (float)softcap.value_or(0.);
  a.scale = scale_of(scale, Dk);
  a.q = c.q.data_ptr(), a.q_stride_b = c.q.stride(0), a.q_stride_n = c.q.stride(1), a.q_stride_h = c.q.stride(2);
  a.k = c.k.data_ptr(), a.k_stride_b = c.k.stride(0), a.k_stride_n = c.k.stride(1), a.k_stride_h = c.k.stride(2);
  a.v = c.v.data_ptr(), a.v_stride_b = c.v.stride(0), a.v_stride_n = c.v.stride(1), a.v_stride_h = c.v.stride(2);
  if (c.starts.defined()) a.starts = c.starts.data_ptr<int32_t>(), a.ends = c.ends.data_ptr<int32_t>();
  a.dev_status = status_of(q);
  a.impl = impl;
}

// keep_low: also what out's rounding left over (16-bit types), for the backward.
std::tuple<Tensor, Tensor, OptTensor> causal_forward(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& seq,
                                          const OptTensor& starts, const OptTensor& ends, std::optional<double> softcap,
                                          std::optional<double> scale, int impl, bool keep_low) {
  Causal c;
  causal_args(c, q, k, v, seq, starts, ends, softcap, scale, impl);
  for (const Tensor* t : {&q, &k, &v}) no_tangent(*t);
  Call call(q);
  Tensor out = at::empty({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options());
  Tensor lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
  c.a.out = out.data_ptr(), c.a.lse = lse.data_ptr<float>();
  Tensor low;
  if (keep_low && q.scalar_type() != at::kFloat) {
    low = at::empty(out.sizes(), out.options());
    c.a.out_low = low.data_ptr();
  }
  done(tc_causal_fwd(&c.a, call.stream), "tc_causal_fwd");
  return {out, lse, low.defined() ? OptTensor(low) : std::nullopt};
}

std::tuple<Tensor, Tensor, Tensor> causal_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out0,
                                                   const OptTensor& low0, const Tensor& lse0, const Tensor& dout0,
                                                   const OptTensor& dlse0,
                                                   const OptTensor& seq, const OptTensor& starts, const OptTensor& ends,
                                                   std::optional<double> softcap, std::optional<double> scale, int impl) {
  Causal c;
  causal_args(c, q, k, v, seq, starts, ends, softcap, scale, impl);
  const int64_t B = q.size(0), N = q.size(1), Hq = q.size(2);
  const at::IntArrayRef rows = q.sizes().slice(0, 3);
  CHECK_VALUE(out0.dim() == 4 && out0.sizes().slice(0, 3) == rows && out0.size(3) == v.size(3) &&
                        out0.scalar_type() == q.scalar_type(),
                    "out shape ", out0.sizes(), " ", out0.scalar_type(), " != [", B, ", ", N, ", ", Hq, ", ", v.size(3), "] ",
                    q.scalar_type());
  CHECK_VALUE(dout0.sizes() == out0.sizes() && dout0.scalar_type() == out0.scalar_type(), "dout shape ", dout0.sizes(),
                    " ", dout0.scalar_type(), " must match out ", out0.sizes(), " ", out0.scalar_type());
  CHECK_VALUE(lse0.sizes() == rows && lse0.scalar_type() == at::kFloat, "lse must be float32 [B, N, Hq]");
  CHECK_VALUE(!dlse0 || (dlse0->sizes() == rows && dlse0->is_floating_point()), "dlse must be floating [", B, ", ", N,
                    ", ", Hq, "], got ", dlse0 ? dlse0->sizes() : rows);
  CHECK_VALUE(!low0 || (low0->sizes() == out0.sizes() && low0->scalar_type() == out0.scalar_type()), "out_low ",
              low0 ? low0->sizes() : rows, " must match out ", out0.sizes());
  same_device(q, out0);
  if (low0) same_device(q, *low0);
  same_device(q, dout0);
  same_device(q, lse0);
  if (dlse0) same_device(q, *dlse0);
  Call call(q);
  const Tensor out = out0.contiguous(), lse = lse0.contiguous(), dout = dout0.contiguous();
  Tensor dlse, low;
  if (dlse0) dlse = table(*dlse0);
  if (low0) low = low0->contiguous();
  Tensor delta = at::empty(rows, q.options().dtype(at::kFloat));
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), q.options()), dv = at::empty(v.sizes(), q.options());
  c.a.lse = lse.data_ptr<float>(), c.a.o = out.data_ptr(), c.a.o_low = low.defined() ? low.data_ptr() : nullptr, c.a.dout = dout.data_ptr();
  c.a.dlse = dlse.defined() ? dlse.data_ptr<float>() : nullptr;
  c.a.delta = delta.data_ptr<float>(), c.a.dq = dq.data_ptr(), c.a.dk = dk.data_ptr(), c.a.dv = dv.data_ptr();
  done(tc_causal_bwd(&c.a, call.stream), "tc_causal_bwd");
  return {dq, dk, dv};
}

// ---------------------------------------------------------------------------
// 8-bit cache
// ---------------------------------------------------------------------------
struct Cache {  // the tensors of a KVCache, checked
  const Tensor &k, &v, &k_scale, &v_scale, &lengths;
  tc_kv_cache c{};
  Cache(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& len, int store)
      : k(k), v(v), k_scale(ks), v_scale(vs), lengths(len) {
    CHECK_VALUE(k.dim() == 4 && v.dim() == 4 && k.sizes().slice(0, 3) == v.sizes().slice(0, 3), "cache k ", k.sizes(),
                      " and v ", v.sizes(), " must be [rows, Hkv, capacity, D]");
    CHECK_VALUE(k.scalar_type() == at::kByte && v.scalar_type() == at::kByte && ks.scalar_type() == at::kFloat &&
                          vs.scalar_type() == at::kFloat && len.scalar_type() == at::kInt,
                      "cache codes must be uint8, scales float32 and lengths int32");
    CHECK_VALUE(ks.sizes() == k.sizes().slice(0, 3) && vs.sizes() == ks.sizes() && len.dim() == 1 && len.size(0) == k.size(0),
                      "cache scales must be [rows, Hkv, capacity] and lengths [rows]");
    CHECK_VALUE(k.is_contiguous() && v.is_contiguous() && ks.is_contiguous() && vs.is_contiguous() && len.is_contiguous(),
                      "cache tensors must be contiguous");
    cuda(k);
    for (const Tensor* t : {&v, &ks, &vs, &len}) same_device(k, *t);
    c.rows = i32(k.size(0), "rows"), c.Hkv = i32(k.size(1), "heads"), c.capacity = i32(k.size(2), "capacity");
    c.Dk = i32(k.size(3), "head dim"), c.Dv = i32(v.size(3), "head dim"), c.store = store;
    c.k = k.data_ptr<uint8_t>(), c.v = v.data_ptr<uint8_t>();
    c.k_scale = ks.data_ptr<float>(), c.v_scale = vs.data_ptr<float>(), c.lengths = len.data_ptr<int32_t>();
  }
};

void kv_write(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs, const Tensor& clen, int store,
              const Tensor& k0, const Tensor& v0, const OptTensor& seq_idx, bool fresh) {
  Cache cache(ck, cv, cks, cvs, clen, store);
  CHECK_VALUE(k0.dim() == 4 && v0.dim() == 4 && k0.sizes().slice(0, 3) == v0.sizes().slice(0, 3) &&
                        k0.scalar_type() == v0.scalar_type(),
                    "k ", k0.sizes(), " ", k0.scalar_type(), " and v ", v0.sizes(), " ", v0.scalar_type(), " do not go together");
  const int64_t B = k0.size(0), N = k0.size(1);
  CHECK_VALUE(k0.size(2) == cache.c.Hkv && k0.size(3) == cache.c.Dk && v0.size(3) == cache.c.Dv, "k ", k0.sizes(), ", v ",
                    v0.sizes(), " do not fit the cache's ", cache.c.Hkv, " heads of ", cache.c.Dk, ", ", cache.c.Dv);
  CHECK_VALUE(seq_idx || B <= cache.c.rows, "batch of ", B, " into a cache of ", cache.c.rows, " rows");
  same_device(ck, k0);
  same_device(ck, v0);
  Tensor ids, starts, ends;
  if (seq_idx) {
    CHECK_VALUE(seq_idx->dim() == 2 && seq_idx->size(0) == B && seq_idx->size(1) == N && integral(*seq_idx),
                      "seq_idx must be an integer tensor [", B, ", ", N, "], got ", seq_idx->sizes(), " ", seq_idx->scalar_type());
    same_device(ck, *seq_idx);
    if (B * N == 0) return;  // names no row
  }
  Call call(k0);
  if (seq_idx) {
    ids = indices(*seq_idx);
    std::tie(starts, ends) = segment_bounds(ids);
  }
  const Tensor k = dense_head(k0), v = dense_head(v0);
  tc_kv_write_args a{};
  a.B = i32(B, "batch"), a.N = i32(N, "length"), a.dtype = dtype_code(k.scalar_type()), a.fresh = fresh;
  a.k = k.data_ptr(), a.k_stride_b = k.stride(0), a.k_stride_n = k.stride(1), a.k_stride_h = k.stride(2);
  a.v = v.data_ptr(), a.v_stride_b = v.stride(0), a.v_stride_n = v.stride(1), a.v_stride_h = v.stride(2);
  if (ids.defined()) a.seq_idx = ids.data_ptr<int32_t>(), a.starts = starts.data_ptr<int32_t>();
  a.dev_status = status_of(k);
  done(tc_kv_write(&cache.c, &a, call.stream), "tc_kv_write");
}

std::tuple<Tensor, Tensor> kv_read(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs, const Tensor& clen,
                                   int store, int64_t length, at::ScalarType dtype) {
  Cache cache(ck, cv, cks, cvs, clen, store);
  CHECK_VALUE(0 <= length && length <= cache.c.capacity, "length ", length, " outside [0, ", cache.c.capacity, "]");
  Call call(ck);
  const int dt = dtype_code(dtype);
  Tensor k = at::empty({cache.c.rows, length, cache.c.Hkv, cache.c.Dk}, ck.options().dtype(dtype));
  Tensor v = at::empty({cache.c.rows, length, cache.c.Hkv, cache.c.Dv}, ck.options().dtype(dtype));
  if (k.numel()) done(tc_kv_read(&cache.c, (int32_t)length, dt, k.data_ptr(), v.data_ptr(), call.stream), "tc_kv_read");
  return {k, v};
}

// Workspace of the split attention: scratch, and arrival counts that are zero
// between calls.  One per device and stream, since calls on one stream run in
// order; not freed, for the process may end after the CUDA context.  A captured call
// replays on any stream, next to any other, so it takes both from the graph's memory:
// scratch of its own, and counts for the calls of its capture on its stream, which
// the graph clears where the first of them was recorded.
struct Work {
  Tensor scratch, counts;
  unsigned long long capture;  // counts: of this capture
};
Work workspace(const Tensor& on, cudaStream_t stream, int64_t floats, int64_t counts) {
  static auto* eager = new std::map<std::pair<int, cudaStream_t>, Work>;
  static auto* captured = new std::map<std::pair<int, cudaStream_t>, Work>;
  const auto f32 = on.options().dtype(at::kFloat), i32 = on.options().dtype(at::kInt);
  const std::pair<int, cudaStream_t> key{on.device().index(), stream};
  cudaStreamCaptureStatus status;
  unsigned long long id = 0;
  CHECK_RUN(cudaStreamGetCaptureInfo(stream, &status, &id) == cudaSuccess, "cached attention: the stream's state is not known");
  if (status != cudaStreamCaptureStatusNone) {
    Work& w = (*captured)[key];
    if (!w.counts.defined() || w.capture != id || w.counts.numel() < counts) {
      w.counts = at::empty({std::max<int64_t>(counts, 4096)}, i32);
      w.capture = id;
      CHECK_RUN(cudaMemsetAsync(w.counts.data_ptr(), 0, w.counts.nbytes(), stream) == cudaSuccess,
                "cached attention: clearing the arrival counts failed");
    }
    return {at::empty({floats}, f32), w.counts, id};
  }
  Work& w = (*eager)[key];
  if (!w.scratch.defined() || w.scratch.numel() < floats)
    w.scratch = at::empty({w.scratch.defined() ? std::max(floats, 2 * w.scratch.numel()) : floats}, f32);
  if (!w.counts.defined() || w.counts.numel() < counts)
    w.counts = at::zeros({std::max<int64_t>(counts, w.counts.defined() ? 2 * w.counts.numel() : 4096)}, i32);
  return w;
}

std::tuple<Tensor, Tensor, OptTensor, OptTensor> kv_attend(const Tensor& ck, const Tensor& cv, const Tensor& cks,
                                                           const Tensor& cvs, const Tensor& clen, int store,
                                                           at::ScalarType cache_dtype, int64_t max_length, const Tensor& q0,
                                                           const OptTensor& k0, const OptTensor& v0, const OptTensor& cos0,
                                                           const OptTensor& sin0, bool interleaved, std::optional<double> softcap,
                                                           std::optional<double> scale, bool advance, bool stored) {
  Cache cache(ck, cv, cks, cvs, clen, store);
  const tc_kv_cache& c = cache.c;
  CHECK_VALUE(q0.dim() == 4 && q0.size(1) == 1, "q_t must be [B, 1, Hq, Dk], got ", q0.sizes());
  const int64_t B = q0.size(0), Hq = q0.size(2), Dk = q0.size(3);
  CHECK_VALUE(Dk == c.Dk && B <= c.rows, "q_t ", q0.sizes(), " incompatible with the cache's ", c.rows, " rows, ", c.Hkv,
                    " heads of ", c.Dk);
  CHECK_VALUE(Hq % c.Hkv == 0 && Hq > 0, "Hq=", Hq, " must be divisible by Hkv=", c.Hkv, ".");
  check_softcap(softcap);
  same_device(ck, q0);
  no_tangent(q0);
  tc_kv_attend_args a{};
  const bool step = k0.has_value();
  if (step) {
    CHECK_VALUE(k0->dim() == 4 && v0->dim() == 4 && k0->size(0) == B && k0->size(1) == 1 &&
                          k0->sizes().slice(0, 3) == v0->sizes().slice(0, 3),
                      "q_t ", q0.sizes(), ", k_t ", k0->sizes(), ", v_t ", v0->sizes(), " do not go together");
    CHECK_VALUE(q0.scalar_type() == k0->scalar_type() && q0.scalar_type() == v0->scalar_type(),
                      "q_t, k_t, v_t must share a dtype, got ", q0.scalar_type(), ", ", k0->scalar_type(), ", ", v0->scalar_type());
    CHECK_VALUE(k0->size(2) == c.Hkv && k0->size(3) == c.Dk && v0->size(3) == c.Dv, "k_t ", k0->sizes(), ", v_t ",
                      v0->sizes(), " do not fit the cache");
    CHECK_VALUE(cos0.has_value() == sin0.has_value(), "rope_cos and rope_sin go together");
    if (cos0) {
      CHECK_VALUE(cos0->dim() == 2 && cos0->sizes() == sin0->sizes() && 2 * cos0->size(1) <= Dk, "rope tables ",
                        cos0->sizes(), ", ", sin0->sizes(), " must be [n_pos, R / 2] with R <= ", Dk);
      CHECK_VALUE(cos0->size(0) > max_length, "rope tables cover ", cos0->size(0), " positions; the token may be at ",
                        max_length);
      same_device(ck, *cos0);
      same_device(ck, *sin0);
    }
    CHECK_VALUE(max_length < c.capacity, "a row may be full: max_length ", max_length, ", capacity ", c.capacity);
    same_device(ck, *k0);
    same_device(ck, *v0);
    no_tangent(*k0);
    no_tangent(*v0);
  }
  Call call(q0);
  const Tensor q = dense_head(q0);
  Tensor out = at::empty({B, 1, Hq, c.Dv}, q.options()), lse = at::empty({B, 1, Hq}, q.options().dtype(at::kFloat));
  Tensor k, v, cos, sin, k_new, v_new;
  a.B = i32(B, "batch"), a.Hq = i32(Hq, "heads"), a.dtype = dtype_code(q.scalar_type());
  a.max_tokens = (int32_t)std::min<int64_t>(max_length + (step ? 1 : 0), c.capacity);
  a.q = q.data_ptr(), a.q_stride_b = q.stride(0), a.q_stride_h = q.stride(2);
  a.has_softcap = softcap.has_value(), a.softcap = (float)softcap.value_or(1.);
  a.scale = scale_of(scale, Dk);
  a.out = out.data_ptr(), a.lse = lse.data_ptr<float>(), a.dev_status = status_of(q);
  if (step) {
    k = dense_head(*k0), v = dense_head(*v0);
    a.k_t = k.data_ptr(), a.k_stride_b = k.stride(0), a.k_stride_h = k.stride(2);
    a.v_t = v.data_ptr(), a.v_stride_b = v.stride(0), a.v_stride_h = v.stride(2);
    if (cos0) {
      cos = table(*cos0), sin = table(*sin0);
      a.rope_cos = cos.data_ptr<float>(), a.rope_sin = sin.data_ptr<float>();
      a.R = (int32_t)(2 * cos.size(1)), a.n_pos = i32(cos.size(0), "table length"), a.interleaved = interleaved;
    }
    a.advance = advance;
    if (stored) {
      k_new = at::empty({B, 1, c.Hkv, c.Dk}, q.options().dtype(cache_dtype));
      v_new = at::empty({B, 1, c.Hkv, c.Dv}, q.options().dtype(cache_dtype));
      a.k_new = k_new.data_ptr(), a.v_new = v_new.data_ptr(), a.new_dtype = dtype_code(cache_dtype);
    }
  }
  const int64_t floats = tc_kv_attend_scratch_floats(&c, a.B, a.Hq, a.max_tokens);
  const int64_t counts = B * (c.Hkv * ((Hq / c.Hkv + 7) / 8) + 1);
  Work w;
  if (B > 0 && floats >= 0 && (floats > 0 || (step && advance))) {
    w = workspace(q, call.stream, floats, counts);
    a.scratch = w.scratch.data_ptr<float>(), a.scratch_floats = w.scratch.numel();
    a.counters = w.counts.data_ptr<int32_t>(), a.num_counters = w.counts.numel();
  }
  done(tc_kv_attend(&c, &a, call.stream), "tc_kv_attend");
  return {out, lse, stored && step ? OptTensor(k_new) : std::nullopt, stored && step ? OptTensor(v_new) : std::nullopt};
}

}  // namespace

PYBIND11_MODULE(_full_attention, m) {
  m.def("set_status", &set_status);
  m.def("rotary", &rotary);
  m.def("segment_bounds", &segment_bounds);
  m.def("causal_forward", &causal_forward);
  m.def("causal_backward", &causal_backward);
  m.def("kv_write", &kv_write);
  m.def("kv_read", &kv_read);
  m.def("kv_attend", &kv_attend);
}
