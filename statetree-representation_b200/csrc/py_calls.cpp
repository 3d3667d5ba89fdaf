// The host path of a module call in native code: TreeLinear products and lists of them (q / k / v, gate / up) for inputs that need
// no conversion, the launches of a matrix's conversion and its check, and the calls of the 8-bit KV pages.  What Python does for such a product (checks, the output
// and its views, pointer arrays, the ctypes call) takes 15 to 30 us, several times a small product's time on the GPU; this takes
// 3 to 5.
//
// Nothing is kept between calls but the addresses of the kernel library's entry points.  A call that is not of the plain form
// (another device or type, a bias, rows that are not contiguous or not 16-byte aligned) returns None and takes the general path in
// linear.py, which also raises its errors.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/version.h>

#include <cstdint>
#include <map>
#include <optional>
#include <stdexcept>
#include <string>
#include <type_traits>
#include <vector>

#include "../../include/statetree_b200.h"

namespace py = pybind11;

namespace {
// the entry points of the loaded kernel library, with the types of the header that this file was compiled with
struct Library {
  decltype(&st_gemv) gemv;
  decltype(&st_gemm) gemm;
  decltype(&st_gemv_list) gemv_list;
  decltype(&st_gemm_list) gemm_list;
  decltype(&st_last_error) last_error;
  decltype(&st_encode) encode;
  decltype(&st_encode_offsets_workspace_bytes) offsets_bytes;
  decltype(&st_encode_offsets) offsets;
  decltype(&st_encode_lists) lists;
  decltype(&st_dec_check) dec_check;
  decltype(&st_lists_check) lists_check;
  decltype(&st_kv8_append) kv8_append;
  decltype(&st_kv8_dequant_blocks) kv8_dequant;
  decltype(&st_kv8_attn_table) kv8_attn;
  decltype(&st_kv8_chunk_attn_table) kv8_chunk;
  decltype(&st_kv8_attn_workspace_bytes) kv8_workspace;
};

// rows of x if it can be read as it is: BF16 [..., N] on `device`, contiguous, 16-byte aligned, at least one row; else 0
int64_t plain_rows(const at::Tensor& x, int64_t N, const at::Device& device) {
  if (x.scalar_type() != at::kBFloat16 || x.device() != device || x.dim() < 1 || x.size(-1) != N || x.numel() == 0 ||
      x.layout() != at::kStrided || !x.is_contiguous() || x.is_conj() || x.is_neg())
    return 0;
  return (reinterpret_cast<uintptr_t>(x.const_data_ptr()) & 15u) == 0 ? x.numel() / N : 0;
}

bool on(const at::Device& device, const at::Tensor& a, const at::Tensor& b, const at::Tensor& c) {
  return a.device() == device && b.device() == device && c.device() == device;
}

void check(const Library& lib, int rc) {
  if (rc != 0) throw std::runtime_error(lib.last_error());
}

std::vector<int64_t> out_sizes(const at::Tensor& x, int64_t M) {
  auto s = x.sizes().vec();
  s.back() = M;
  return s;
}

// binds the entry points: their addresses by name
Library library(const std::map<std::string, uint64_t>& address) {
  Library lib;
  auto bind = [&](auto& entry, const char* name) {
    entry = reinterpret_cast<std::remove_reference_t<decltype(entry)>>(address.at(name));
  };
  bind(lib.gemv, "st_gemv");
  bind(lib.gemm, "st_gemm");
  bind(lib.gemv_list, "st_gemv_list");
  bind(lib.gemm_list, "st_gemm_list");
  bind(lib.last_error, "st_last_error");
  bind(lib.encode, "st_encode");
  bind(lib.offsets_bytes, "st_encode_offsets_workspace_bytes");
  bind(lib.offsets, "st_encode_offsets");
  bind(lib.lists, "st_encode_lists");
  bind(lib.dec_check, "st_dec_check");
  bind(lib.lists_check, "st_lists_check");
  bind(lib.kv8_append, "st_kv8_append");
  bind(lib.kv8_dequant, "st_kv8_dequant_blocks");
  bind(lib.kv8_attn, "st_kv8_attn_table");
  bind(lib.kv8_chunk, "st_kv8_chunk_attn_table");
  bind(lib.kv8_workspace, "st_kv8_attn_workspace_bytes");
  return lib;
}

// x W^T for one tree: the GEMV (use_gemm false) or the tcgen05 GEMM
py::object linear(const Library& lib, bool use_gemm, const at::Tensor& tree, const at::Tensor& eo, const at::Tensor& el,
                  const at::Tensor& eb, const at::Tensor& x, const at::Tensor& ws, const at::Tensor& cnt) {
  const int64_t M = tree.size(0) * 16, N = tree.size(1) * 64, B = plain_rows(x, N, tree.device());
  if (B == 0 || !on(tree.device(), eo, el, eb)) return py::none();
  at::Tensor y;
  int rc;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(tree.device());
    y = at::empty(out_sizes(x, M), x.options().requires_grad(false));
    void* stream = c10::cuda::getCurrentCUDAStream(tree.device().index()).stream();
    const int64_t ws_bytes = ws.numel() * (int64_t)ws.element_size();
    auto i32 = [](const at::Tensor& t) { return reinterpret_cast<const int32_t*>(t.const_data_ptr()); };
    auto u32 = [](const at::Tensor& t) { return reinterpret_cast<const uint32_t*>(t.const_data_ptr()); };
    int32_t* const c = reinterpret_cast<int32_t*>(cnt.data_ptr());
    rc = use_gemm ? lib.gemm(tree.const_data_ptr(), i32(eo), u32(el), x.const_data_ptr(), y.data_ptr(), nullptr, B, M, N,
                             ws.data_ptr(), ws_bytes, c, stream)
                  : lib.gemv(tree.const_data_ptr(), i32(eo), u32(eb), u32(el), x.const_data_ptr(), y.data_ptr(), nullptr, B, M, N,
                             ws.data_ptr(), ws_bytes, c, stream);
  }
  check(lib, rc);
  return py::cast(y);
}

// the same for one to four trees that share their columns; tables = (eo, el, eb) of each.  ws (GEMV) or cnt (GEMM)
py::object linear_list(const Library& lib, bool use_gemm, const std::vector<at::Tensor>& trees,
                       const std::vector<std::vector<at::Tensor>>& tables, const at::Tensor& x, const at::Tensor& scratch) {
  constexpr int MAX = 4;
  const int n = (int)trees.size();
  if (n < 1 || n > MAX || tables.size() != trees.size()) return py::none();
  const at::Device device = trees[0].device();
  const int64_t N = trees[0].size(1) * 64, B = plain_rows(x, N, device);
  if (B == 0) return py::none();
  for (int i = 0; i < n; ++i)
    if (trees[i].device() != device || trees[i].size(1) * 64 != N || tables[i].size() != 3 ||
        !on(device, tables[i][0], tables[i][1], tables[i][2]))
      return py::none();
  std::vector<at::Tensor> ys;
  int rc;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(device);
    const void* T[MAX];
    const int32_t* EO[MAX];
    const uint32_t *EL[MAX], *EB[MAX];
    void* Y[MAX];
    int64_t M[MAX], total = 0;
    for (int i = 0; i < n; ++i) total += M[i] = trees[i].size(0) * 16;
    at::Tensor flat = at::empty({B * total}, x.options().requires_grad(false));
    int64_t at_row = 0;
    for (int i = 0; i < n; ++i) {                                // one allocation, a contiguous [.., M] block per tree
      auto sizes = out_sizes(x, M[i]);
      std::vector<int64_t> strides(sizes.size());
      int64_t step = 1;
      for (int d = (int)sizes.size() - 1; d >= 0; --d) { strides[d] = step; step *= sizes[d]; }
      ys.push_back(flat.as_strided(sizes, strides, B * at_row));
      at_row += M[i];
      T[i] = trees[i].const_data_ptr();
      EO[i] = reinterpret_cast<const int32_t*>(tables[i][0].const_data_ptr());
      EL[i] = reinterpret_cast<const uint32_t*>(tables[i][1].const_data_ptr());
      EB[i] = reinterpret_cast<const uint32_t*>(tables[i][2].const_data_ptr());
      Y[i] = ys[i].data_ptr();
    }
    void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    rc = use_gemm ? lib.gemm_list(n, T, EO, EL, x.const_data_ptr(), Y, nullptr, B, M, N, reinterpret_cast<int32_t*>(scratch.data_ptr()),
                                  stream)
                  : lib.gemv_list(n, T, EO, EB, EL, x.const_data_ptr(), Y, nullptr, B, M, N, scratch.data_ptr(),
                                  scratch.numel() * (int64_t)scratch.element_size(), stream);
  }
  check(lib, rc);
  return py::cast(ys);
}

// W [M, N] BF16 on a GPU, contiguous, 16-byte aligned -> (tree, rows, cols, bits, eo, el, eb): the format's parts and the kernels'
// side tables.  The lists' length depends on the data, so the stream is synchronised once, before they are made; the kernel that
// fills them may still run when the call returns.
py::tuple encode(const Library& lib, const at::Tensor& W) {
  TORCH_CHECK(W.is_cuda() && W.dim() == 2 && W.scalar_type() == at::kBFloat16 && W.is_contiguous(),
              "encode: a contiguous BF16 matrix on a GPU");
  const int64_t M = W.size(0), N = W.size(1);
  TORCH_CHECK(M > 0 && N > 0 && M % 16 == 0 && N % 64 == 0, "encode: rows must be a multiple of 16, columns of 64");
  const int64_t NG = N / 64, nrec = M / 16 * NG;
  at::Tensor tree, rows, cols, bits, eo, el, eb;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(W.device());
    void* stream = c10::cuda::getCurrentCUDAStream(W.device().index()).stream();
    const auto u8 = W.options().requires_grad(false).dtype(at::kByte), i32 = u8.dtype(at::kInt);
    auto ip = [](const at::Tensor& t) { return reinterpret_cast<int32_t*>(t.data_ptr()); };
    auto up = [](const at::Tensor& t) { return reinterpret_cast<uint32_t*>(t.data_ptr()); };
    tree = at::empty({M / 16, NG, 1552}, u8);
    eo = at::empty({nrec + 1}, i32);
    eb = at::empty({M / 16 * ((NG + 7) / 8), 16}, i32);
    const int64_t need = lib.offsets_bytes(M, N);
    at::Tensor rowcnt = at::empty({M * NG}, u8), reccnt = at::empty({nrec + 1}, i32), roff = at::empty({M * NG}, i32),
               ws = at::empty({need}, u8);
    uint8_t* const rc = reinterpret_cast<uint8_t*>(rowcnt.data_ptr());
    check(lib, lib.encode(W.const_data_ptr(), M, N, tree.data_ptr(), rc, ip(reccnt), stream));
    check(lib, lib.offsets(rc, ip(reccnt), M, N, ip(roff), ip(eo), ws.data_ptr(), need, stream));
    const int64_t n = eo.select(0, nrec).item<int32_t>();         // (synchronises)
    rows = at::empty({n}, i32);
    cols = at::empty({n}, i32);
    bits = at::empty({n}, i32.dtype(at::kShort));
    el = n ? at::empty({n}, i32) : at::zeros({1}, i32);
    void* const spare = el.data_ptr();                            // (no escapes: empty tensors have no address; nothing is written)
    check(lib, lib.lists(W.const_data_ptr(), M, N, rc, ip(roff), ip(eo), up(el), up(eb),
                         reinterpret_cast<int32_t*>(n ? rows.data_ptr() : spare), reinterpret_cast<int32_t*>(n ? cols.data_ptr() : spare),
                         reinterpret_cast<int16_t*>(n ? bits.data_ptr() : spare), stream));
  }
  return py::make_tuple(tree, rows, cols, bits, eo, el, eb);
}

// launches the check of a tree against W (contiguous, 16-byte aligned) and of the stored lists and eb, if there are any (an empty
// vector: none): an int32 count of what is wrong, on the GPU
at::Tensor check_start(const Library& lib, const at::Tensor& tree, const at::Tensor& eo, const at::Tensor& el, const at::Tensor& W,
                       const std::vector<at::Tensor>& stored) {
  TORCH_CHECK(W.is_cuda() && W.dim() == 2 && W.scalar_type() == at::kBFloat16 && W.is_contiguous(),
              "dec_check: a contiguous BF16 matrix on a GPU");
  TORCH_CHECK(tree.is_cuda() && tree.dim() == 3 && tree.size(0) * 16 == W.size(0) && tree.size(1) * 64 == W.size(1),
              "dec_check: the tree is not one of this matrix");
  TORCH_CHECK(eo.is_cuda() && el.is_cuda() && (stored.empty() || stored.size() == 4), "dec_check: tables");
  py::gil_scoped_release nogil;
  const int64_t M = W.size(0), N = W.size(1);
  const c10::cuda::CUDAGuard guard(W.device());
  void* stream = c10::cuda::getCurrentCUDAStream(W.device().index()).stream();
  at::Tensor bad = at::zeros({1}, W.options().requires_grad(false).dtype(at::kInt));
  auto i32 = [](const at::Tensor& t) { return reinterpret_cast<const int32_t*>(t.const_data_ptr()); };
  auto u32 = [](const at::Tensor& t) { return reinterpret_cast<const uint32_t*>(t.const_data_ptr()); };
  int32_t* const b = reinterpret_cast<int32_t*>(bad.data_ptr());
  check(lib, lib.dec_check(tree.const_data_ptr(), i32(eo), u32(el), M, N, W.const_data_ptr(), b, stream));
  if (!stored.empty()) {
    for (const at::Tensor& t : stored) TORCH_CHECK(t.is_cuda(), "dec_check: tables");
    const int64_t n = stored[0].numel();
    TORCH_CHECK(stored[1].numel() == n && stored[2].numel() == n, "dec_check: lists of different lengths");
    check(lib, lib.lists_check(i32(stored[0]), i32(stored[1]), reinterpret_cast<const int16_t*>(stored[2].const_data_ptr()), n, i32(eo),
                               u32(el), u32(stored[3]), M, N, W.const_data_ptr(), b, stream));
  }
  return bad;
}
// ---- 8-bit KV pages.  Each returns None where the call is not of the plain form (the checks in ops.py then say what is wrong with it)
using Maybe = std::optional<at::Tensor>;
constexpr int64_t PAGE = 16;

bool flat(const at::Tensor& t, at::ScalarType type, const at::Device& device) {
  return t.scalar_type() == type && t.device() == device && t.layout() == at::kStrided && t.is_contiguous();
}
// pages uint8 [blocks, H, 2, 16, D] and exps int8 [blocks, H, 2] on a GPU
bool pages8(const at::Tensor& pages, const at::Tensor& exps) {
  return pages.is_cuda() && pages.dim() == 5 && pages.size(2) == 2 && pages.size(3) == PAGE && (pages.size(4) == 64 || pages.size(4) == 128) &&
         flat(pages, at::kByte, pages.device()) && flat(exps, at::kChar, pages.device()) && exps.dim() == 3 && exps.size(0) == pages.size(0) &&
         exps.size(1) == pages.size(1) && exps.size(2) == 2;
}
// BF16 [N, heads, D], heads contiguous, as the kernels' 16-byte vectors need it
bool rows8(const at::Tensor& t, int64_t D, const at::Device& device) {
  return t.scalar_type() == at::kBFloat16 && t.device() == device && t.layout() == at::kStrided && t.dim() == 3 && t.size(2) == D &&
         t.numel() > 0 && t.stride(2) == 1 && (t.stride(1) == D || t.size(1) == 1) && t.stride(0) % 8 == 0 && !t.is_conj() && !t.is_neg() &&
         (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0;
}
bool norm8(const Maybe& w, int64_t D, const at::Device& device) {
  return !w || (flat(*w, at::kBFloat16, device) && w->numel() == D && (reinterpret_cast<uintptr_t>(w->const_data_ptr()) & 15u) == 0);
}
template <typename T>
const T* of(const Maybe& t) { return t ? reinterpret_cast<const T*>(t->const_data_ptr()) : nullptr; }
template <typename T>
const T* of(const at::Tensor& t) { return reinterpret_cast<const T*>(t.const_data_ptr()); }

// append; returns the rotated queries (True without any)
py::object kv8_append(const Library& lib, const at::Tensor& pages, const at::Tensor& exps, const at::Tensor& marks, const at::Tensor& bad,
                      const at::Tensor& K, const at::Tensor& V, const at::Tensor& slots, const Maybe& positions, const Maybe& cos,
                      const Maybe& sin, bool interleaved, const Maybe& q, const Maybe& q_norm, const Maybe& k_norm, double eps,
                      const Maybe& q_out) {
  if (!pages8(pages, exps)) return py::none();
  const at::Device device = pages.device();
  const int64_t H = pages.size(1), D = pages.size(4);
  if (!rows8(K, D, device) || !rows8(V, D, device)) return py::none();
  const int64_t N = K.size(0);
  if (K.size(1) != H || V.size(0) != N || V.size(1) != H || !flat(slots, at::kLong, device) || slots.numel() != N ||
      !flat(marks, at::kInt, device) || marks.numel() < 17 * pages.size(0) || !flat(bad, at::kInt, device) || bad.numel() < 1 ||
      !norm8(k_norm, D, device) || !norm8(q_norm, D, device) || cos.has_value() != sin.has_value())
    return py::none();
  int64_t step = 0, span = 0;
  if (cos) {
    if (!positions || !flat(*positions, at::kLong, device) || (positions->numel() != N && positions->numel() != 1) || !flat(*cos, at::kFloat, device) ||
        !flat(*sin, at::kFloat, device) || cos->dim() != 2 || sin->sizes() != cos->sizes() || cos->size(1) != D / 2 || cos->size(0) < 1)
      return py::none();
    step = positions->numel() > 1;
    span = cos->size(0);
  }
  if (q && (!rows8(*q, D, device) || q->size(0) != N)) return py::none();
  if (q_out && (!q || !rows8(*q_out, D, device) || q_out->sizes() != q->sizes())) return py::none();
  at::Tensor out;
  int rc;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(device);
    if (q) out = q_out ? *q_out : at::empty(q->sizes(), q->options().requires_grad(false));
    void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    rc = lib.kv8_append(K.const_data_ptr(), V.const_data_ptr(), K.stride(0), V.stride(0), of<int64_t>(slots), N, H, D, pages.data_ptr(),
                        reinterpret_cast<int8_t*>(exps.data_ptr()), pages.size(0), cos ? of<int64_t>(positions) : nullptr, step,
                        of<float>(cos), of<float>(sin), span, interleaved ? 1 : 0, of<void>(k_norm), of<void>(q), q ? q->stride(0) : 0,
                        of<void>(q_norm), q ? q->size(1) : 0, q ? out.data_ptr() : nullptr, q ? out.stride(0) : 0, eps,
                        reinterpret_cast<int32_t*>(marks.data_ptr()), reinterpret_cast<int32_t*>(bad.data_ptr()), stream);
  }
  check(lib, rc);
  return q ? py::cast(out) : py::cast(true);
}

// attention of one query per sequence (chunk false) or of cu's rows (chunk true; cu None: one each)
py::object kv8_attention(const Library& lib, bool chunk, const at::Tensor& pages, const at::Tensor& exps, const at::Tensor& q,
                         const Maybe& cu, const at::Tensor& table, const at::Tensor& lens, double scale, int64_t splits,
                         const Maybe& starts, int64_t min_pages, const Maybe& given, int64_t window) {
  if (!pages8(pages, exps)) return py::none();
  const at::Device device = pages.device();
  const int64_t H = pages.size(1), D = pages.size(4);
  if (!rows8(q, D, device) || table.dim() != 2) return py::none();
  const int64_t T = q.size(0), Hq = q.size(1), B = table.size(0);
  if (Hq % H || B < 1 || table.scalar_type() != at::kInt || table.device() != device || table.layout() != at::kStrided || table.stride(1) != 1 ||
      !flat(lens, at::kInt, device) || lens.numel() != B || (starts && (!flat(*starts, at::kInt, device) || starts->numel() != B)) ||
      splits < 1 || window < 0 || (cu ? !flat(*cu, at::kInt, device) || cu->numel() != B + 1 : T != B))
    return py::none();
  if (given && (!rows8(*given, D, device) || given->sizes() != q.sizes())) return py::none();
  at::Tensor out, ws;
  int rc;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(device);
    out = given ? *given : at::empty(q.sizes(), q.options().requires_grad(false));
    float *wo = nullptr, *wml = nullptr;
    if (const int64_t need = lib.kv8_workspace(T, B, Hq, H, D, splits, chunk)) {      // partial results of this call alone
      ws = at::empty({need / 4}, q.options().requires_grad(false).dtype(at::kFloat));
      wo = reinterpret_cast<float*>(ws.data_ptr());
      wml = wo + T * Hq * splits * D;
    }
    void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    rc = chunk ? lib.kv8_chunk(q.const_data_ptr(), q.stride(0), T, Hq, of<int32_t>(cu), B, pages.const_data_ptr(), of<int8_t>(exps),
                               pages.size(0), H, D, of<int32_t>(table), table.size(1), table.stride(0), of<int32_t>(lens),
                               of<int32_t>(starts), window, out.data_ptr(), out.stride(0), wo, wml, scale, splits, stream)
               : lib.kv8_attn(q.const_data_ptr(), q.stride(0), B, Hq, pages.const_data_ptr(), of<int8_t>(exps), pages.size(0), H, D,
                              of<int32_t>(table), table.size(1), table.stride(0), of<int32_t>(lens), of<int32_t>(starts), window, out.data_ptr(),
                              out.stride(0), wo, wml, scale, splits, min_pages, stream);
  }
  check(lib, rc);
  return py::cast(out);
}

// listed pages (None: all) as dense BF16 [n, 16, H, D]
py::object kv8_dense(const Library& lib, const at::Tensor& pages, const at::Tensor& exps, const Maybe& blocks) {
  if (!pages8(pages, exps) || (blocks && (!flat(*blocks, at::kInt, pages.device()) || blocks->dim() != 1))) return py::none();
  const int64_t H = pages.size(1), D = pages.size(4), n = blocks ? blocks->numel() : pages.size(0);
  at::Tensor K, V;
  int rc;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(pages.device());
    K = at::empty({n, PAGE, H, D}, pages.options().requires_grad(false).dtype(at::kBFloat16));
    V = at::empty_like(K);
    rc = lib.kv8_dequant(pages.const_data_ptr(), of<int8_t>(exps), pages.size(0), H, D, of<int32_t>(blocks), n, K.data_ptr(), V.data_ptr(),
                         c10::cuda::getCurrentCUDAStream(pages.device().index()).stream());
  }
  check(lib, rc);
  return py::make_tuple(K, V);
}
}  // namespace

PYBIND11_MODULE(_calls, m) {
  m.attr("ABI") = ST_ABI_VERSION;                // what this file was compiled against (compared when it is loaded)
  m.attr("TORCH") = TORCH_VERSION;
  py::class_<Library>(m, "Library");
  m.def("library", &library);
  m.def("linear", &linear);
  m.def("linear_list", &linear_list);
  m.def("encode", &encode);
  m.def("check_start", &check_start);
  m.def("kv8_append", &kv8_append);
  m.def("kv8_attention", &kv8_attention);
  m.def("kv8_dense", &kv8_dense);
}
