// torch bindings of the linear layers on 4-bit weights (include/qe_mx.h), registered in qengine_amd._C by
// bindings.cpp. As there: every op writes into the caller's tensors, enqueues on the current stream of their
// device, never syncs or allocates, and raises RuntimeError for arguments outside its contract. The _check_*
// functions run the same validation without the device requirement and without a launch.
#include "bindings_util.hpp"
#include "mx_form.hpp"
#include "qe_mx.h"

namespace {

using Opt = c10::optional<torch::Tensor>;

constexpr int64_t LD_END = 1 << 23;

// A row argument of `w` columns (0: any): its own row stride, the width for a single row, whose stride is of no
// account. An output's rows must not overlap.
Rows mx_rows(const torch::Tensor& t, torch::ScalarType dt, const char* name, int64_t n, int64_t w, bool dev) {
  TORCH_CHECK(t.scalar_type() == dt, name, " has wrong dtype ", t.scalar_type());
  TORCH_CHECK(!dev || t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.dim() == 1 || t.dim() == 2, name, " must be [n, w] (or one row)");
  const int64_t rows = t.dim() == 1 ? 1 : t.size(0), width = t.size(-1);
  TORCH_CHECK(width <= 1 || t.stride(-1) == 1, name, " must have unit inner stride");
  TORCH_CHECK(rows >= 1 && rows <= QE_MX_MAX_ROWS, name, " must have 1..2^24 rows");
  TORCH_CHECK(n == 0 || rows == n, name, " must have ", n, " rows, got ", rows);
  TORCH_CHECK(w == 0 || width == w, name, " must be ", w, " wide, got ", width);
  TORCH_CHECK(width >= 1, name, " has no columns");
  const int64_t ld = rows == 1 ? width : t.stride(0);
  TORCH_CHECK(ld >= width, name, " rows must not overlap");
  TORCH_CHECK(ld < LD_END, name, ": row strides must be below 2^23");
  return {(int)rows, (long)width, (long)ld};
}

void mx_width(int64_t K, const char* name) {
  TORCH_CHECK(K >= 1 && K <= QE_MX_MAX_WIDTH, name, ": widths are 1..2^20");
}

// 8-bit rows: codes (float8_e4m3fn, or uint8) and scale codes (float8_e8m0fnu, or uint8).
struct Mx8 {
  Rows q, s;
};
Mx8 parse_mx8(const torch::Tensor& q, const torch::Tensor& s, int64_t n, int64_t K, bool dev) {
  const int64_t blocks = K ? (K + 31) / 32 : 0;
  TORCH_CHECK(q.scalar_type() == torch::kFloat8_e4m3fn || q.scalar_type() == torch::kByte,
              "q must be float8_e4m3fn (or uint8 codes), got ", q.scalar_type());
  TORCH_CHECK(s.scalar_type() == torch::kFloat8_e8m0fnu || s.scalar_type() == torch::kByte,
              "s must be float8_e8m0fnu (or uint8 codes), got ", s.scalar_type());
  const Rows Q = mx_rows(q, q.scalar_type(), "q", n, blocks * 32, dev);
  TORCH_CHECK(Q.w % 32 == 0, "q must be a multiple of 32 wide");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 && Q.ld % 16 == 0,
              "q must be 16-byte aligned rows");
  return {Q, mx_rows(s, s.scalar_type(), "s", Q.n, Q.w / 32, dev)};
}

void one_device(const torch::Tensor& t, std::initializer_list<const torch::Tensor*> others) {
  for (const auto* o : others) TORCH_CHECK(o->device() == t.device(), "arguments must be on one device");
}

void parse_mx4(const torch::Tensor& wq, int64_t N, int64_t K, bool dev) {
  chk(wq, torch::kByte, "wq", dev);
  mx_width(K, "wq");
  TORCH_CHECK(N >= 1 && N <= QE_MX_MAX_ROWS, "weights have 1..2^24 rows");
  TORCH_CHECK((size_t)wq.numel() == qe_mx4_bytes((int)N, (int)K), "wq must hold mx4_bytes(", N, ", ", K, ") = ",
              qe_mx4_bytes((int)N, (int)K), " bytes, has ", wq.numel());
  TORCH_CHECK(reinterpret_cast<uintptr_t>(wq.data_ptr()) % 16 == 0, "wq must be 16-byte aligned");
}

// -------------------------------------------------------------------------------- weights
Rows parse_weight(const torch::Tensor& w, const torch::Tensor& wq, const char* name, bool dev) {
  TORCH_CHECK(w.dim() == 2, name, " must be [N, K]");
  const Rows W = mx_rows(w, BF, name, 0, 0, dev);
  parse_mx4(wq, W.n, W.w, dev);
  one_device(w, {&wq});
  return W;
}
void mx4_quant(torch::Tensor w, torch::Tensor wq) {
  const Rows W = parse_weight(w, wq, "w", true);
  const c10::DeviceGuard guard(w.device());
  raise_on(qe_mx4_quant(w.data_ptr(), W.ld, wq.data_ptr(), W.n, (int)W.w, stream_of(w)), "qe_mx4_quant");
}
void mx4_dequant(torch::Tensor wq, torch::Tensor out) {
  const Rows O = parse_weight(out, wq, "out", true);
  const c10::DeviceGuard guard(out.device());
  raise_on(qe_mx4_dequant(wq.data_ptr(), out.data_ptr(), O.ld, O.n, (int)O.w, stream_of(out)), "qe_mx4_dequant");
}

// -------------------------------------------------------------------------------- rows
struct ActArgs {
  Rows x;
  Mx8 o;
  int K;
};
ActArgs parse_act(const torch::Tensor& x, const torch::Tensor& q, const torch::Tensor& s, bool glu, bool dev) {
  const Rows X = mx_rows(x, BF, glu ? "gu" : "x", 0, 0, dev);
  TORCH_CHECK(!glu || X.w % 2 == 0, "gu must hold [gate | up] rows");
  const int64_t K = glu ? X.w / 2 : X.w;
  mx_width(K, glu ? "gu" : "x");
  one_device(x, {&q, &s});
  return {X, parse_mx8(q, s, X.n, K, dev), (int)K};
}
void quant_mx8(torch::Tensor x, torch::Tensor q, torch::Tensor s) {
  const auto a = parse_act(x, q, s, false, true);
  const c10::DeviceGuard guard(x.device());
  raise_on(qe_quant_mx8(x.data_ptr(), a.x.ld, q.data_ptr(), a.o.q.ld, s.data_ptr(), a.o.s.ld, a.x.n, a.K,
                        stream_of(x)),
           "qe_quant_mx8");
}
void swiglu_mx8(torch::Tensor gu, torch::Tensor q, torch::Tensor s) {
  const auto a = parse_act(gu, q, s, true, true);
  const c10::DeviceGuard guard(gu.device());
  raise_on(qe_swiglu_mx8(gu.data_ptr(), a.x.ld, q.data_ptr(), a.o.q.ld, s.data_ptr(), a.o.s.ld, a.x.n, a.K,
                         stream_of(gu)),
           "qe_swiglu_mx8");
}

struct NormArgs {
  Rows x, d, sum;
  Mx8 o;
};
NormArgs parse_norm(const torch::Tensor& x, const Opt& delta, const torch::Tensor& w, const torch::Tensor& q,
                    const torch::Tensor& s, const Opt& sum, bool dev) {
  const Rows X = mx_rows(x, BF, "x", 0, 0, dev);
  mx_width(X.w, "x");
  chk(w, BF, "w", dev);
  TORCH_CHECK(w.numel() == X.w, "w must have x's width");
  TORCH_CHECK(delta.has_value() || !sum.has_value(), "sum needs delta");
  one_device(x, {&w, &q, &s});
  NormArgs a{X, {0, 0, 0}, {0, 0, 0}, parse_mx8(q, s, X.n, X.w, dev)};
  if (delta.has_value()) {
    a.d = mx_rows(*delta, BF, "delta", X.n, X.w, dev);
    a.sum = sum.has_value() ? mx_rows(*sum, BF, "sum", X.n, X.w, dev) : X;
    one_device(x, {&*delta});
    if (sum.has_value()) one_device(x, {&*sum});
  }
  return a;
}
void rmsnorm1p_mx8(torch::Tensor x, Opt delta, torch::Tensor w, torch::Tensor q, torch::Tensor s, double eps,
                   Opt sum) {
  const auto a = parse_norm(x, delta, w, q, s, sum, true);
  const c10::DeviceGuard guard(x.device());
  void* to = !delta.has_value() ? nullptr : sum.has_value() ? sum->data_ptr() : x.data_ptr();
  raise_on(qe_rmsnorm1p_mx8(x.data_ptr(), a.x.ld, delta.has_value() ? delta->data_ptr() : nullptr, a.d.ld,
                            w.data_ptr(), to, a.sum.ld, q.data_ptr(), a.o.q.ld, s.data_ptr(), a.o.s.ld, a.x.n,
                            (int)a.x.w, (float)eps, stream_of(x)),
           "qe_rmsnorm1p_mx8");
}

// -------------------------------------------------------------------------------- product
struct GemmArgs {
  Mx8 x;
  Rows o;
  void* ws;
  size_t ws_bytes;
};
GemmArgs parse_gemm(const torch::Tensor& wq, const torch::Tensor& xq, const torch::Tensor& xs,
                    const torch::Tensor& out, const Opt& ws, bool dev) {
  const Mx8 X = parse_mx8(xq, xs, 0, 0, dev);
  mx_width(X.q.w, "q");
  const Rows O = mx_rows(out, BF, "out", X.q.n, 0, dev);
  parse_mx4(wq, O.w, X.q.w, dev);
  one_device(out, {&wq, &xq, &xs});
  GemmArgs a{X, O, nullptr, 0};
  if (ws.has_value() && ws->numel() > 0) {
    chk(*ws, torch::kByte, "ws", dev);
    TORCH_CHECK(reinterpret_cast<uintptr_t>(ws->data_ptr()) % 16 == 0, "ws must be 16-byte aligned");
    one_device(out, {&*ws});
    a.ws = ws->data_ptr();
    a.ws_bytes = (size_t)ws->numel();
  }
  return a;
}
void gemm_mx4(torch::Tensor wq, torch::Tensor xq, torch::Tensor xs, torch::Tensor out, Opt ws) {
  const auto a = parse_gemm(wq, xq, xs, out, ws, true);
  const c10::DeviceGuard guard(out.device());
  raise_on(qe_gemm_mx4(wq.data_ptr(), xq.data_ptr(), a.x.q.ld, xs.data_ptr(), a.x.s.ld, out.data_ptr(), a.o.ld,
                       a.o.n, (int)a.o.w, (int)a.x.q.w, a.ws, a.ws_bytes, stream_of(out)),
           "qe_gemm_mx4");
}

// A given kernel, for the tests of each at any size.
void gemm_mx4_as(int64_t kernel, int64_t splits, torch::Tensor wq, torch::Tensor xq, torch::Tensor xs,
                 torch::Tensor out, Opt ws) {
  auto a = parse_gemm(wq, xq, xs, out, ws, false);
  TORCH_CHECK(kernel >= -1 && kernel < 16 && splits >= 1 && splits <= 64 &&
                  qe::mx::gemm_form_ok((int)kernel, (int)splits, a.o.n, (int)a.o.w, (int)a.x.q.w, a.ws_bytes),
              "kernel ", kernel, " does not take this call in ", splits, " splits");
  a = parse_gemm(wq, xq, xs, out, ws, true);
  const c10::DeviceGuard guard(out.device());
  raise_on(qe::mx::gemm_as((int)kernel, (int)splits,
                           {wq.data_ptr(), xq.data_ptr(), a.x.q.ld, xs.data_ptr(), a.x.s.ld, out.data_ptr(), a.o.ld,
                            a.o.n, (int)a.o.w, (int)a.x.q.w, a.ws, a.ws_bytes},
                           stream_of(out)),
           "gemm_mx4");
}

int64_t positive(int64_t v, int64_t most, const char* what) {
  TORCH_CHECK(v >= 1 && v <= most, what, " must be 1..", most, ", got ", v);
  return v;
}

}  // namespace

void bind_mx(py::module_& m) {
  m.def("mx4_bytes",
        [](int64_t N, int64_t K) {
          return (int64_t)qe_mx4_bytes((int)positive(N, QE_MX_MAX_ROWS, "N"), (int)positive(K, QE_MX_MAX_WIDTH, "K"));
        },
        py::arg("N"), py::arg("K"), "bytes of an [N, K] weight in microscaled 4-bit floating point");
  m.def("mx4_ws_bytes",
        [](int64_t n, int64_t N, int64_t K) {
          return (int64_t)qe_gemm_mx4_ws_size((int)positive(n, QE_MX_MAX_ROWS, "n"),
                                              (int)positive(N, QE_MX_MAX_ROWS, "N"),
                                              (int)positive(K, QE_MX_MAX_WIDTH, "K"));
        },
        py::arg("n"), py::arg("N"), py::arg("K"), "bytes of gemm_mx4's workspace for n rows");
  m.def("mx4_quant", &mx4_quant, py::arg("w"), py::arg("wq"), "wq = w [N, K] as 4-bit codes with scales");
  m.def("mx4_dequant", &mx4_dequant, py::arg("wq"), py::arg("out"), "out [N, K] = the values of a 4-bit weight");
  m.def("quant_mx8", &quant_mx8, py::arg("x"), py::arg("q"), py::arg("s"), "rows as 8-bit codes with scales");
  m.def("swiglu_mx8", &swiglu_mx8, py::arg("gu"), py::arg("q"), py::arg("s"),
        "silu(gate) * up of gu = [gate | up] as 8-bit codes with scales");
  m.def("rmsnorm1p_mx8", &rmsnorm1p_mx8, py::arg("x"), py::arg("delta"), py::arg("w"), py::arg("q"), py::arg("s"),
        py::arg("eps"), py::arg("sum") = py::none(),
        "rmsnorm1p whose output is 8-bit codes with scales; bf16(x + delta) goes to sum (default: x)");
  m.def("gemm_mx4", &gemm_mx4, py::arg("wq"), py::arg("xq"), py::arg("xs"), py::arg("out"),
        py::arg("ws") = py::none(), "out [n, N] = 8-bit rows [n, K] @ (4-bit weight [N, K])^T");
  m.def("_check_mx4_weight", [](torch::Tensor w, torch::Tensor wq) {
    const Rows W = parse_weight(w, wq, "w", false);
    return std::vector<int64_t>{W.n, W.w, W.ld};
  });
  m.def("_check_act_mx8", [](torch::Tensor x, torch::Tensor q, torch::Tensor s, bool glu) {
    const auto a = parse_act(x, q, s, glu, false);
    return std::vector<int64_t>{a.x.n, a.K, a.x.ld, a.o.q.ld, a.o.s.ld};
  });
  m.def("_check_rmsnorm1p_mx8", [](torch::Tensor x, Opt d, torch::Tensor w, torch::Tensor q, torch::Tensor s,
                                   Opt sum) {
    const auto a = parse_norm(x, d, w, q, s, sum, false);
    return std::vector<int64_t>{a.x.n, a.x.w, a.x.ld, a.d.ld, a.sum.ld, a.o.q.ld, a.o.s.ld};
  });
  m.def("_check_gemm_mx4", [](torch::Tensor wq, torch::Tensor xq, torch::Tensor xs, torch::Tensor out, Opt ws) {
    const auto a = parse_gemm(wq, xq, xs, out, ws, false);
    return std::vector<int64_t>{a.o.n, a.o.w, a.x.q.w, a.x.q.ld, a.x.s.ld, a.o.ld};
  });
  // how gemm_mx4 runs a call (host only): (kernel, splits, weight rows of that, kernel and splits of the others)
  m.def("_gemm_mx4_form", [](int64_t n, int64_t N, int64_t K, int64_t ws_bytes) {
    TORCH_CHECK(ws_bytes >= 0 && K % 32 == 0, "K is a multiple of 32, a workspace has no negative size");
    const auto f = qe::mx::gemm_form((int)positive(n, QE_MX_MAX_ROWS, "n"), (int)positive(N, QE_MX_MAX_ROWS, "N"),
                                     (int)positive(K, QE_MX_MAX_WIDTH, "K"), (size_t)ws_bytes);
    return std::make_tuple(f.kernel, f.splits, f.cut, f.rest_kernel, f.rest_splits);
  });
  m.def("_gemm_mx4_as", &gemm_mx4_as);
}
