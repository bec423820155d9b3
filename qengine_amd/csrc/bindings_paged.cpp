// torch bindings of the paged KV cache (include/qe_paged.h), registered in qengine_amd._C by bindings.cpp.
// As there: every op writes into the caller's tensors, enqueues on the current stream of their device, never
// syncs or allocates, and raises RuntimeError for arguments outside its contract. The _check_* functions run
// the same validation without the device requirement and without a launch.
#include "bindings_util.hpp"
#include "qe_paged.h"

namespace qe {
namespace paged {
void decode_form(int B, int Hkv, int cap, int NS, int window, int sinks, int (&form)[3]);  // attn_paged.hip
}
}  // namespace qe

namespace {

void same_device(const torch::Tensor& t, std::initializer_list<const torch::Tensor*> others) {
  for (const auto* o : others) TORCH_CHECK(o->device() == t.device(), "arguments must be on one device");
}

// A pool pair [N, Hkv, P, 256] (lead = 0) or [layers, N, Hkv, P, 256] (lead = 1, where layers may be left out).
struct Pool {
  int layers, N, Hkv, P;
  size_t page_bytes;
};
Pool parse_pool(const torch::Tensor& kp, const torch::Tensor& vp, bool kv8, bool lead, bool dev) {
  if (kv8) {
    chk_kv8(kp, "kp", dev);
    chk_kv8(vp, "vp", dev);
  } else {
    chk(kp, BF, "kp", dev);
    chk(vp, BF, "vp", dev);
  }
  const int d = (int)kp.dim();
  TORCH_CHECK((d == 4 || (lead && d == 5)) && kp.size(-1) == HD && vp.sizes() == kp.sizes(),
              "kp/vp must be ", lead ? "[(layers,) N, Hkv, P, 256]" : "[N, Hkv, P, 256]", " with equal sizes");
  const int64_t L = d == 5 ? kp.size(0) : 1, N = kp.size(-4), H = kp.size(-3), P = kp.size(-2);
  TORCH_CHECK(L >= 1 && L <= 65535 && N >= 1 && N <= (1 << 24) && H >= 1 && H <= 16384,
              "pools need 1..65535 layers, 1..2^24 pages and at least one head");
  TORCH_CHECK(P >= 16 && P <= 32768 && (P & (P - 1)) == 0, "the page size must be a power of two, 16..32768");
  chk16(kp, HD, "kp");
  chk16(vp, HD, "vp");
  return {(int)L, (int)N, (int)H, (int)P, (size_t)(H * P * HD) * kp.element_size()};
}

// The page table [B, M] (rows any stride apart, or one row).
struct Table {
  int B, M;
  long ld;
};
Table parse_table(const torch::Tensor& t, int64_t P, bool dev) {
  TORCH_CHECK((!dev || t.is_cuda()) && t.scalar_type() == I32, "table must be int32 on the GPU");
  TORCH_CHECK(t.dim() == 2 && t.size(0) >= 1 && t.size(0) <= QE_PAGED_MAX_SEQS && t.size(1) >= 1,
              "table must be [B, M], B in 1..", QE_PAGED_MAX_SEQS, ", M >= 1");
  TORCH_CHECK(t.size(1) == 1 || t.stride(1) == 1, "table must have unit inner stride");
  const long B = t.size(0), M = t.size(1), ld = B == 1 ? M : (long)t.stride(0);
  TORCH_CHECK(ld >= M, "table rows must not overlap");
  TORCH_CHECK(P >= 16 && P <= 32768 && (P & (P - 1)) == 0, "the page size must be a power of two, 16..32768");
  TORCH_CHECK(M * P <= (1 << 23) - 64, "a table row holds at most 2^23 - 64 positions");
  return {(int)B, (int)M, ld};
}

void chk_ints(const torch::Tensor& t, int64_t n, const char* name, bool dev) {
  chk(t, I32, name, dev);
  TORCH_CHECK(t.numel() == n, name, " must have ", n, " elements, got ", t.numel());
}

// Rows of a batch: n = B * R. One row's stride is of no account.
Rows batch_rows(const torch::Tensor& t, const char* name, bool dev) {
  Rows r = rows(t, BF, name, dev);
  if (r.n == 1) r.ld = r.w;
  TORCH_CHECK(r.n == 0 || r.ld >= r.w, name, " rows must not overlap");
  return r;
}

struct DecodeArgs {
  Pool p;
  Table t;
  int R, Hq, NS;
  long ldp, ldo;
};
DecodeArgs parse_decode(const torch::Tensor& q, const torch::Tensor& kp, const torch::Tensor& vp,
                        const torch::Tensor& table, const torch::Tensor& pos, const torch::Tensor& qg,
                        const torch::Tensor& part_o, const torch::Tensor& part_ml, const torch::Tensor& out,
                        int64_t window, int64_t sinks, bool kv8, bool dev) {
  const auto Q = batch_rows(q, "q", dev), G = batch_rows(qg, "qg", dev), O = batch_rows(out, "out", dev);
  const auto p = parse_pool(kp, vp, kv8, false, dev);
  const auto t = parse_table(table, p.P, dev);
  chk_ints(pos, t.B, "pos", dev);
  chk(part_o, F32, "part_o", dev);
  chk(part_ml, F32, "part_ml", dev);
  TORCH_CHECK(Q.n >= t.B && Q.n <= 8l * t.B && Q.n % t.B == 0,
              "decode takes 1..8 rows per sequence: q must have B * R rows");
  const long Hq = Q.w / HD;
  TORCH_CHECK(Hq >= 1 && Q.w == Hq * HD && Q.ld == Q.w && Hq % p.Hkv == 0 && Hq <= 65535,
              "q rows must be contiguous and Hq*256 wide, Hq % Hkv == 0");
  TORCH_CHECK(G.n == Q.n && O.n == Q.n && G.w == Hq * 2 * HD && O.w == Q.w,
              "qg and out must have q's rows; qg width Hq*512; out width Hq*256");
  chk16(q, Q.ld, "q");
  TORCH_CHECK(part_o.dim() == 4 && part_o.size(0) >= Q.n && part_o.size(1) == Hq && part_o.size(2) >= 1 &&
                  part_o.size(2) <= 65535 && part_o.size(3) == HD,
              "part_o must be [>= B*R, Hq, NS, 256]");
  TORCH_CHECK(part_ml.numel() == part_o.numel() / HD * 2, "part_ml must be [>= B*R, Hq, NS, 2]");
  chk16(part_o, HD, "part_o");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(part_ml.data_ptr()) % 8 == 0, "part_ml must be 8-byte aligned");
  const int NS = (int)part_o.size(2);
  TORCH_CHECK(window >= 0 && window < (1 << 23) && sinks >= 0, "window must be 0..2^23-1, sinks >= 0");
  TORCH_CHECK(window == 0 || NS >= 4, "a window needs at least 4 splits");
  TORCH_CHECK((long)t.B * p.Hkv * NS <= 0x3fffffffL, "B * Hkv * NS must be below 2^30");
  if (dev) same_device(q, {&kp, &vp, &table, &pos, &qg, &part_o, &part_ml, &out});
  return {p, t, (int)(Q.n / t.B), (int)Hq, NS, G.ld, O.ld};
}
int sinks_of(int64_t sinks) { return (int)std::min<int64_t>(sinks, 1 << 23); }

void attn_decode_paged(torch::Tensor q, torch::Tensor kp, torch::Tensor vp, torch::Tensor table,
                       torch::Tensor pos, torch::Tensor qg, torch::Tensor part_o, torch::Tensor part_ml,
                       torch::Tensor out, int64_t window, int64_t sinks) {
  const auto a = parse_decode(q, kp, vp, table, pos, qg, part_o, part_ml, out, window, sinks, false, true);
  const c10::DeviceGuard guard(q.device());
  raise_on(qe_attn_decode_paged(q.data_ptr(), kp.data_ptr(), vp.data_ptr(), table.data_ptr<int>(), a.t.ld,
                                pos.data_ptr<int>(), qg.data_ptr(), a.ldp, part_o.data_ptr<float>(),
                                part_ml.data_ptr<float>(), out.data_ptr(), a.ldo, a.t.B, a.R, a.Hq,
                                a.p.Hkv, a.p.N, a.p.P, a.t.M, a.NS, (int)window, sinks_of(sinks),
                                1.0f / 16.0f, stream_of(q)),
           "qe_attn_decode_paged");
}

void attn_decode_paged_fp8(torch::Tensor q, torch::Tensor kp, torch::Tensor vp, torch::Tensor table,
                           torch::Tensor pos, torch::Tensor qg, torch::Tensor part_o,
                           torch::Tensor part_ml, torch::Tensor out, double k_scale, double v_scale,
                           int64_t window, int64_t sinks) {
  kv_scales(k_scale, v_scale);
  const auto a = parse_decode(q, kp, vp, table, pos, qg, part_o, part_ml, out, window, sinks, true, true);
  const c10::DeviceGuard guard(q.device());
  raise_on(qe_attn_decode_paged_fp8(q.data_ptr(), kp.data_ptr(), vp.data_ptr(), table.data_ptr<int>(),
                                    a.t.ld, pos.data_ptr<int>(), qg.data_ptr(), a.ldp,
                                    part_o.data_ptr<float>(), part_ml.data_ptr<float>(), out.data_ptr(),
                                    a.ldo, a.t.B, a.R, a.Hq, a.p.Hkv, a.p.N, a.p.P, a.t.M, a.NS,
                                    (int)window, sinks_of(sinks), 1.0f / 16.0f, (float)k_scale,
                                    (float)v_scale, stream_of(q)),
           "qe_attn_decode_paged_fp8");
}

struct PrepArgs {
  Pool p;
  Table t;
  int R, Hq, rd;
  long ldp;
};
PrepArgs parse_prep(const torch::Tensor& qg, const torch::Tensor& k, const torch::Tensor& v,
                    const torch::Tensor& qnw, const torch::Tensor& knw, const torch::Tensor& inv_freq,
                    const torch::Tensor& pos, const torch::Tensor& q_out, const torch::Tensor& kp,
                    const torch::Tensor& vp, const torch::Tensor& table, bool kv8, bool dev) {
  // (input rows may overlap: they are only read)
  const auto G = rows(qg, BF, "qg", dev), K = rows(k, BF, "k", dev), V = rows(v, BF, "v", dev);
  const auto Q = batch_rows(q_out, "q_out", dev);
  TORCH_CHECK(G.n == 1 || (G.ld == K.ld && G.ld == V.ld), "qg/k/v must share a row stride");
  TORCH_CHECK(G.ld >= 1, "qg must have a positive row stride");
  chk(qnw, BF, "qnw", dev);
  chk(knw, BF, "knw", dev);
  chk(inv_freq, F32, "inv_freq", dev);
  const auto p = parse_pool(kp, vp, kv8, false, dev);
  const auto t = parse_table(table, p.P, dev);
  chk_ints(pos, t.B, "pos", dev);
  TORCH_CHECK(G.n >= t.B && G.n <= 65535 && G.n % t.B == 0 && K.n == G.n && V.n == G.n && Q.n == G.n &&
                  Q.ld == Q.w,
              "prep takes B * R rows (at most 65535), equal in every argument, and contiguous q_out rows");
  const long Hq = Q.w / HD;
  TORCH_CHECK(Hq >= 1 && Q.w == Hq * HD && Hq + p.Hkv <= 16384, "q_out width must be Hq*256");
  TORCH_CHECK(G.w == Hq * 2 * HD && K.w == (long)p.Hkv * HD && V.w == (long)p.Hkv * HD,
              "row widths must be qg = Hq*512, k = v = Hkv*256");
  TORCH_CHECK(qnw.numel() == HD && knw.numel() == HD, "qnw/knw must have 256 elements");
  TORCH_CHECK(inv_freq.numel() >= 1 && inv_freq.numel() * 2 <= HD,
              "rotary dims (2 * inv_freq.numel()) must be 2..256");
  if (dev) same_device(qg, {&k, &v, &qnw, &knw, &inv_freq, &pos, &q_out, &kp, &vp, &table});
  return {p, t, G.n / t.B, (int)Hq, (int)inv_freq.numel() * 2, G.ld};
}

void attn_prep_paged(torch::Tensor qg, torch::Tensor k, torch::Tensor v, torch::Tensor qnw,
                     torch::Tensor knw, torch::Tensor inv_freq, torch::Tensor pos, torch::Tensor q_out,
                     torch::Tensor kp, torch::Tensor vp, torch::Tensor table, double eps) {
  const auto a = parse_prep(qg, k, v, qnw, knw, inv_freq, pos, q_out, kp, vp, table, false, true);
  const c10::DeviceGuard guard(qg.device());
  raise_on(qe_attn_prep_paged(qg.data_ptr(), k.data_ptr(), v.data_ptr(), a.ldp, qnw.data_ptr(),
                              knw.data_ptr(), inv_freq.data_ptr<float>(), pos.data_ptr<int>(),
                              q_out.data_ptr(), kp.data_ptr(), vp.data_ptr(), table.data_ptr<int>(),
                              a.t.ld, a.t.B, a.R, a.Hq, a.p.Hkv, a.p.N, a.p.P, a.t.M, a.rd, (float)eps,
                              stream_of(qg)),
           "qe_attn_prep_paged");
}

void attn_prep_paged_fp8(torch::Tensor qg, torch::Tensor k, torch::Tensor v, torch::Tensor qnw,
                         torch::Tensor knw, torch::Tensor inv_freq, torch::Tensor pos, torch::Tensor q_out,
                         torch::Tensor kp, torch::Tensor vp, torch::Tensor table, double eps,
                         double k_scale, double v_scale) {
  kv_scales(k_scale, v_scale);
  const auto a = parse_prep(qg, k, v, qnw, knw, inv_freq, pos, q_out, kp, vp, table, true, true);
  const c10::DeviceGuard guard(qg.device());
  raise_on(qe_attn_prep_paged_fp8(qg.data_ptr(), k.data_ptr(), v.data_ptr(), a.ldp, qnw.data_ptr(),
                                  knw.data_ptr(), inv_freq.data_ptr<float>(), pos.data_ptr<int>(),
                                  q_out.data_ptr(), kp.data_ptr(), vp.data_ptr(), table.data_ptr<int>(),
                                  a.t.ld, a.t.B, a.R, a.Hq, a.p.Hkv, a.p.N, a.p.P, a.t.M, a.rd, (float)eps,
                                  (float)k_scale, (float)v_scale, stream_of(qg)),
           "qe_attn_prep_paged_fp8");
}

// ---- operations on pages
int parse_ref(const torch::Tensor& ref, bool dev) {
  chk(ref, I32, "ref", dev);
  TORCH_CHECK(ref.numel() >= 1 && ref.numel() <= (1 << 24), "ref must have one element per page, 1..2^24");
  return (int)ref.numel();
}

Table parse_free(const torch::Tensor& table, const torch::Tensor& ref, const torch::Tensor& first,
                 const torch::Tensor& last, int64_t page, bool dev) {
  const auto t = parse_table(table, page, dev);
  parse_ref(ref, dev);
  chk_ints(first, t.B, "first", dev);
  chk_ints(last, t.B, "last", dev);
  if (dev) same_device(table, {&ref, &first, &last});
  return t;
}
void kv_pages_free(torch::Tensor table, torch::Tensor ref, torch::Tensor first, torch::Tensor last,
                   int64_t page) {
  const auto t = parse_free(table, ref, first, last, page, true);
  const c10::DeviceGuard guard(table.device());
  raise_on(qe_kv_pages_free(table.data_ptr<int>(), t.ld, ref.data_ptr<int>(), first.data_ptr<int>(),
                            last.data_ptr<int>(), t.B, t.M, (int)ref.numel(), (int)page, stream_of(table)),
           "qe_kv_pages_free");
}

Table parse_extend(const torch::Tensor& table, const torch::Tensor& ref, const torch::Tensor& pos,
                   const torch::Tensor& count, int64_t page, const torch::Tensor& missing, bool dev) {
  const auto t = parse_table(table, page, dev);
  parse_ref(ref, dev);
  chk_ints(pos, t.B, "pos", dev);
  chk_ints(count, t.B, "count", dev);
  chk_ints(missing, 1, "missing", dev);
  if (dev) same_device(table, {&ref, &pos, &count, &missing});
  return t;
}
void kv_pages_extend(torch::Tensor table, torch::Tensor ref, torch::Tensor pos, torch::Tensor count,
                     int64_t page, torch::Tensor missing) {
  const auto t = parse_extend(table, ref, pos, count, page, missing, true);
  const c10::DeviceGuard guard(table.device());
  raise_on(qe_kv_pages_extend(table.data_ptr<int>(), t.ld, ref.data_ptr<int>(), pos.data_ptr<int>(),
                              count.data_ptr<int>(), missing.data_ptr<int>(), t.B, t.M, (int)ref.numel(),
                              (int)page, stream_of(table)),
           "qe_kv_pages_extend");
}

bool is_kv8(const torch::Tensor& kp) { return kp.scalar_type() != BF; }

struct MoveArgs {
  Pool p;
  Table t;
  int m;
};
MoveArgs parse_alloc(const torch::Tensor& table, const torch::Tensor& ref, const torch::Tensor& kp,
                     const torch::Tensor& vp, const torch::Tensor& ws, bool dev) {
  const auto p = parse_pool(kp, vp, is_kv8(kp), true, dev);
  const auto t = parse_table(table, p.P, dev);
  TORCH_CHECK(parse_ref(ref, dev) == p.N, "ref must have one element per page of the pools");
  chk(ws, I32, "ws", dev);
  TORCH_CHECK((size_t)ws.numel() * 4 >= qe_kv_pages_ws_size(p.N), "ws must have at least 2 * N + 8 elements");
  if (dev) same_device(table, {&ref, &kp, &vp, &ws});
  return {p, t, 0};
}
MoveArgs parse_fork(const torch::Tensor& table, const torch::Tensor& ref, const torch::Tensor& src,
                    const torch::Tensor& dst, const torch::Tensor& length, const torch::Tensor& kp,
                    const torch::Tensor& vp, const torch::Tensor& missing, const torch::Tensor& ws,
                    bool dev) {
  auto a = parse_alloc(table, ref, kp, vp, ws, dev);
  TORCH_CHECK(src.numel() >= 1 && src.numel() <= 1024, "fork takes 1..1024 pairs");
  a.m = (int)src.numel();
  chk_ints(src, a.m, "src", dev);
  chk_ints(dst, a.m, "dst", dev);
  chk_ints(length, a.m, "length", dev);
  chk_ints(missing, 1, "missing", dev);
  if (dev) same_device(table, {&src, &dst, &length, &missing});
  return a;
}
void kv_pages_fork(torch::Tensor table, torch::Tensor ref, torch::Tensor src, torch::Tensor dst,
                   torch::Tensor length, torch::Tensor kp, torch::Tensor vp, torch::Tensor missing,
                   torch::Tensor ws) {
  const auto a = parse_fork(table, ref, src, dst, length, kp, vp, missing, ws, true);
  const c10::DeviceGuard guard(table.device());
  raise_on(qe_kv_pages_fork(table.data_ptr<int>(), a.t.ld, ref.data_ptr<int>(), src.data_ptr<int>(),
                            dst.data_ptr<int>(), length.data_ptr<int>(), a.m, kp.data_ptr(), vp.data_ptr(),
                            a.p.layers, a.p.page_bytes, missing.data_ptr<int>(), ws.data_ptr(), a.t.B,
                            a.t.M, a.p.N, a.p.P, stream_of(table)),
           "qe_kv_pages_fork");
}

void kv_pages_compact(torch::Tensor table, torch::Tensor ref, torch::Tensor kp, torch::Tensor vp,
                      torch::Tensor ws) {
  const auto a = parse_alloc(table, ref, kp, vp, ws, true);
  const c10::DeviceGuard guard(table.device());
  raise_on(qe_kv_pages_compact(table.data_ptr<int>(), a.t.ld, ref.data_ptr<int>(), kp.data_ptr(),
                               vp.data_ptr(), a.p.layers, a.p.page_bytes, ws.data_ptr(), a.t.B, a.t.M,
                               a.p.N, stream_of(table)),
           "qe_kv_pages_compact");
}

MoveArgs parse_copy(const torch::Tensor& kp, const torch::Tensor& vp, const torch::Tensor& src,
                    const torch::Tensor& dst, bool dev) {
  const auto p = parse_pool(kp, vp, is_kv8(kp), true, dev);
  TORCH_CHECK(src.numel() >= 1 && src.numel() <= 65535, "copy takes 1..65535 pairs");
  const int m = (int)src.numel();
  chk_ints(src, m, "src", dev);
  chk_ints(dst, m, "dst", dev);
  if (dev) same_device(kp, {&vp, &src, &dst});
  return {p, {}, m};
}
void kv_pages_copy(torch::Tensor kp, torch::Tensor vp, torch::Tensor src, torch::Tensor dst) {
  const auto a = parse_copy(kp, vp, src, dst, true);
  const c10::DeviceGuard guard(kp.device());
  raise_on(qe_kv_pages_copy(kp.data_ptr(), vp.data_ptr(), a.p.layers, a.p.page_bytes, src.data_ptr<int>(),
                            dst.data_ptr<int>(), a.m, a.p.N, stream_of(kp)),
           "qe_kv_pages_copy");
}

}  // namespace

void bind_paged(py::module_& m) {
  m.def("attn_decode_paged", &attn_decode_paged, py::arg("q"), py::arg("kp"), py::arg("vp"),
        py::arg("table"), py::arg("pos"), py::arg("qg"), py::arg("part_o"), py::arg("part_ml"),
        py::arg("out"), py::arg("window") = 0, py::arg("sinks") = 0,
        "gated attention of 1..8 rows per sequence over a paged KV cache");
  m.def("attn_decode_paged_fp8", &attn_decode_paged_fp8, py::arg("q"), py::arg("kp"), py::arg("vp"),
        py::arg("table"), py::arg("pos"), py::arg("qg"), py::arg("part_o"), py::arg("part_ml"),
        py::arg("out"), py::arg("k_scale"), py::arg("v_scale"), py::arg("window") = 0,
        py::arg("sinks") = 0, "attn_decode_paged over pools of E4M3FN codes");
  m.def("attn_prep_paged", &attn_prep_paged,
        "q/k norm + RoPE of a batch's new rows, K and V written to pages (qg, k, v, qnw, knw, inv_freq, pos, "
        "q_out, kp, vp, table, eps)");
  m.def("attn_prep_paged_fp8", &attn_prep_paged_fp8,
        "attn_prep_paged into pools of E4M3FN codes (..., eps, k_scale, v_scale)");
  m.def("kv_pages_free", &kv_pages_free,
        "release the pages wholly inside positions [first, last) of each sequence (table, ref, first, last, "
        "page)");
  m.def("kv_pages_extend", &kv_pages_extend,
        "map the pages of positions [pos, pos + count) (table, ref, pos, count, page, missing)");
  m.def("kv_pages_fork", &kv_pages_fork,
        "sequences dst become copies of the first length positions of src (table, ref, src, dst, length, kp, "
        "vp, missing, ws)");
  m.def("kv_pages_compact", &kv_pages_compact,
        "move the pages in use to the lowest ids (table, ref, kp, vp, ws)");
  m.def("kv_pages_copy", &kv_pages_copy, "copy page data src[i] -> dst[i] (kp, vp, src, dst)");
  m.def("_check_attn_decode_paged",
        [](torch::Tensor q, torch::Tensor kp, torch::Tensor vp, torch::Tensor table, torch::Tensor pos,
           torch::Tensor qg, torch::Tensor po, torch::Tensor pml, torch::Tensor out, int64_t window,
           int64_t sinks, bool kv8) {
          const auto a = parse_decode(q, kp, vp, table, pos, qg, po, pml, out, window, sinks, kv8, false);
          return std::vector<int64_t>{a.t.B, a.R, a.Hq, a.p.Hkv, a.p.N, a.p.P, a.t.M, a.NS, a.t.ld, a.ldp,
                                      a.ldo};
        });
  // how the decode cuts a call (host only): (least slice, most slices of a row, persistent waves)
  m.def("_attn_decode_paged_form", [](int B, int Hkv, int cap, int NS, int window, int sinks) {
    TORCH_CHECK(B >= 1 && Hkv >= 1 && cap >= 1 && NS >= 1 && window >= 0 && sinks >= 0, "sizes must be positive");
    int f[3];
    qe::paged::decode_form(B, Hkv, cap, NS, window, window ? std::min(sinks, cap) : 0, f);
    return std::make_tuple(f[0], f[1], f[2] != 0);
  });
  m.def("_check_attn_prep_paged",
        [](torch::Tensor qg, torch::Tensor k, torch::Tensor v, torch::Tensor qnw, torch::Tensor knw,
           torch::Tensor inv_freq, torch::Tensor pos, torch::Tensor q_out, torch::Tensor kp,
           torch::Tensor vp, torch::Tensor table, bool kv8) {
          const auto a = parse_prep(qg, k, v, qnw, knw, inv_freq, pos, q_out, kp, vp, table, kv8, false);
          return std::vector<int64_t>{a.t.B, a.R, a.Hq, a.p.Hkv, a.p.N, a.p.P, a.t.M, a.rd, a.t.ld, a.ldp};
        });
  m.def("_check_kv_pages_free", [](torch::Tensor t, torch::Tensor r, torch::Tensor f, torch::Tensor l,
                                   int64_t page) { parse_free(t, r, f, l, page, false); });
  m.def("_check_kv_pages_extend",
        [](torch::Tensor t, torch::Tensor r, torch::Tensor p, torch::Tensor c, int64_t page,
           torch::Tensor miss) { parse_extend(t, r, p, c, page, miss, false); });
  m.def("_check_kv_pages_fork",
        [](torch::Tensor t, torch::Tensor r, torch::Tensor s, torch::Tensor d, torch::Tensor n,
           torch::Tensor kp, torch::Tensor vp, torch::Tensor miss,
           torch::Tensor ws) { parse_fork(t, r, s, d, n, kp, vp, miss, ws, false); });
  m.def("_check_kv_pages_compact",
        [](torch::Tensor t, torch::Tensor r, torch::Tensor kp, torch::Tensor vp, torch::Tensor ws) {
          parse_alloc(t, r, kp, vp, ws, false);
        });
  m.def("_check_kv_pages_copy", [](torch::Tensor kp, torch::Tensor vp, torch::Tensor s, torch::Tensor d) {
    parse_copy(kp, vp, s, d, false);
  });
}
