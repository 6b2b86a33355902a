// TORCH_LIBRARY(logo_hip) registration of the hot-path entry points of
// liblogo_hip.so, so that torch.library / torch.compile see them as operators
// with schemas (their fake kernels are registered from logo_amd/_torch_ops.py).
//
// Host code only: every operator checks its tensors (device, dtype,
// contiguity, shapes), allocates its outputs with the caching allocator on the
// current stream, and calls the C entry point, which launches on that stream.
// The library's own checks stay the last line (a failure raises with
// logo_last_error()).  Operators, the C entry point each wraps, and the
// reference code it replaces:
//   compact       logo_compact        build_selection, logo/ops/common.py:71-107
//   dense_meta    logo_dense_meta     all-rows metadata of the dense / SWA branches
//   sq_fwd        logo_sq_fwd         logo/ops/selected_full_attn.py:33-121, :340-362
//   sq_bwd_delta  logo_sq_bwd_delta   :124-138, :365-371
//   sq_bwd_dq     logo_sq_bwd_dq      :141-228, :424-432
//   sq_bwd_dkv    logo_sq_bwd_dkv     :231-337, :433-445
//   sq_bwd_dqkv   logo_sq_bwd_dqkv    dq and dk/dv together (one fused pass for
//                                     the sliding window, logo/layers/utils.py:144-147)
//   sq_bwd        delta, then dqkv    :124-445 (dq, dk, dv; workspaces internal)
//   epilogue_fwd  logo_epilogue_fwd   logo/layers/logo.py:180-181, :225-226, :256-258
//   epilogue_bwd  logo_epilogue_bwd   the autograd of epilogue_fwd
//   decode_attn   logo_decode_attn    logo/layers/logo.py:228-249
//   paged_attn    logo_paged_attn     the same over a paged cache, and :183-209 for chunks over it
//   paged_append  logo_paged_append   logo/cache.py:97-118, logo/layers/logo.py:132-150
//   rotary        logo_rotary         logo/modules/rotary.py:58-106
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cstdlib>
#include <initializer_list>
#include <limits>
#include <mutex>
#include <optional>
#include <utility>
#include <vector>

#include "../../include/logo_hip.h"

namespace {

void* sp() { return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream().stream()); }

void ok(int rc, const char* what) { TORCH_CHECK(rc == LOGO_OK, what, " failed: ", logo_last_error()); }

const void* cptr(const at::Tensor& t) { return t.data_ptr(); }
void* mptr(at::Tensor& t) { return t.data_ptr(); }
template <typename T>
const T* opt_ptr(const std::optional<at::Tensor>& t) {
  return t.has_value() ? static_cast<const T*>(t->data_ptr()) : nullptr;
}

void need(const at::Tensor& t, const char* name, at::ScalarType dt) {
  TORCH_CHECK(t.is_cuda(), "logo_hip: ", name, " must be a ROCm GPU tensor");
  TORCH_CHECK(t.scalar_type() == dt, "logo_hip: ", name, " must be ", dt, ", got ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), "logo_hip: ", name, " must be contiguous");
}

// compact(selection bool or u8 [N] or [N, lanes], cu i32 [nseq+1])
//   -> (q_idx i64 [lanes, N], pos i32 [lanes, N], meta)
std::tuple<at::Tensor, at::Tensor, at::Tensor> compact(const at::Tensor& sel, const at::Tensor& cu) {
  need(sel, "selection", sel.scalar_type() == at::kBool ? at::kBool : at::kByte);
  need(cu, "cu_seqlens", at::kInt);
  const int64_t n = sel.size(0);
  const int lanes = sel.dim() == 2 ? (int)sel.size(1) : 1;
  const int nseq = (int)cu.numel() - 1;
  auto i32 = cu.options();
  // entries past each lane's Sq: zero, written by the compaction itself
  // (n == 0 keeps one zero entry per lane)
  auto q_idx = n > 0 ? at::empty({lanes, n}, i32.dtype(at::kLong)) : at::zeros({lanes, 1}, i32.dtype(at::kLong));
  auto pos = n > 0 ? at::empty({lanes, n}, i32) : at::zeros({lanes, 1}, i32);
  auto meta = at::empty({lanes * LOGO_META_STRIDE(nseq)}, i32);
  auto ws = at::empty({(int64_t)logo_compact_workspace_bytes(n, lanes)}, i32.dtype(at::kByte));
  ok(logo_compact(static_cast<const uint8_t*>(sel.data_ptr()), n, lanes, cu.data_ptr<int32_t>(), nseq,
                  q_idx.data_ptr<int64_t>(), pos.data_ptr<int32_t>(), meta.data_ptr<int32_t>(), ws.data_ptr(),
                  sp()),
     "logo_compact");
  return {q_idx, pos, meta};
}

at::Tensor dense_meta(const at::Tensor& cu, int64_t n_tokens) {
  need(cu, "cu_seqlens", at::kInt);
  const int nseq = (int)cu.numel() - 1;
  auto meta = at::empty({LOGO_META_STRIDE(nseq)}, cu.options());
  ok(logo_dense_meta(cu.data_ptr<int32_t>(), nseq, n_tokens, meta.data_ptr<int32_t>(), sp()), "logo_dense_meta");
  return meta;
}

// q, k, v of one element type (bf16; fp16 or fp32 for the C library's
// query-sparse kernels, which rejects other fp16 / fp32 calls itself);
// returns its dtype code.
int check_attn(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  const at::ScalarType qt = q.scalar_type();
  const at::ScalarType dt = qt == at::kHalf || qt == at::kFloat ? qt : at::kBFloat16;
  need(q, "q", dt);
  need(k, "k", dt);
  need(v, "v", dt);
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "logo_hip: q, k, v must be [N, heads, D]");
  TORCH_CHECK(k.size(0) == q.size(0) && v.sizes() == k.sizes() && k.size(2) == q.size(2),
              "logo_hip: q [N, HQ, D], k and v [N, H, D] must agree");
  return dt == at::kHalf ? LOGO_DTYPE_F16 : dt == at::kFloat ? LOGO_DTYPE_F32 : LOGO_DTYPE_BF16;
}

// Whether the call's backward reads q and dO in place (no compacted copies):
// head dim 256 and fp32.
bool generic_path(const at::Tensor& q, int dtype) { return logo_sq_generic((int)q.size(2), dtype) != 0; }

// Split workspace of the fwd, dq and dk/dv kernels for this shape (empty: no
// split).  Calls on one buffer must not overlap, except dk/dv with the dq of
// its own call, whose counters and partials are apart.  The part of fwd and dq
// depends only on the device's CU count, HQ and D (the pieces a split aims for
// fill the device twice, whatever N is): at most 136 MB at D = 128 on MI355X,
// also at D = 256; that of dk/dv, at most 118 MB at D = 128, is there only
// where its key blocks are few enough to be cut.
//  * Outside graph capture: one buffer per (device, stream), kept across
//    calls and grown on demand.  The kernels leave its counter prefix zero,
//    so only a new buffer needs the zero fill, and calls on one stream run in
//    order, so they never overlap on it.  At most kMaxCachedStreams buffers
//    are kept; beyond that the oldest entry is dropped (its memory returns to
//    the caching allocator on its own stream, after the work queued there).
//  * Under capture (hipStreamIsCapturing): a fresh buffer per call from the
//    caching allocator, its counters cleared by a fill kernel recorded in the
//    graph.  The graph's memory pool keeps the buffer for the graph's
//    lifetime, so a later eager call that regrows the cached buffer cannot
//    free memory a replay still uses, and a replay never depends on counters
//    that eager calls left behind.
// The environment variable LOGO_SQ_SPLIT=0 turns the split off (A/B timing,
// and tests that compare kernel variants bit for bit).
constexpr size_t kMaxCachedStreams = 16;

at::Tensor split_workspace(const at::Tensor& q, const at::Tensor& k, const at::Tensor& cu, int dtype, bool fwd) {
  const char* env = std::getenv("LOGO_SQ_SPLIT");
  size_t bytes = 0;
  if (env == nullptr || env[0] != '0') {
    if (!generic_path(q, dtype))
      bytes = logo_sq_kv_workspace_bytes(q.size(0), (int)cu.numel() - 1, (int)q.size(1), (int)k.size(1),
                                         (int)q.size(2));
    else if (dtype != LOGO_DTYPE_F32 && q.size(0) >= 2 * LOGO_WIDE_SPLIT_KEYS &&
             !(fwd && q.size(0) < LOGO_WIDE_FWD_MIN_TOKENS * (cu.numel() - 1)))
      bytes = logo_sq_wide_workspace_bytes((int)q.size(1));
  }
  if (bytes == 0) return at::empty({0}, q.options().dtype(at::kByte));
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  TORCH_CHECK(hipStreamIsCapturing(static_cast<hipStream_t>(sp()), &status) == hipSuccess,
              "logo_hip: hipStreamIsCapturing failed");
  if (status != hipStreamCaptureStatusNone) {
    auto ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    ws.narrow(0, 0, (int64_t)logo_sq_workspace_counter_bytes()).zero_();
    return ws;
  }
  static std::mutex mu;
  static std::vector<std::pair<std::pair<int, void*>, at::Tensor>> cache;  // oldest first
  const auto key = std::make_pair((int)q.get_device(), sp());
  std::lock_guard<std::mutex> lock(mu);
  auto it = std::find_if(cache.begin(), cache.end(), [&](const auto& e) { return e.first == key; });
  if (it == cache.end()) {
    if (cache.size() >= kMaxCachedStreams) cache.erase(cache.begin());
    cache.emplace_back(key, at::Tensor());
    it = cache.end() - 1;
  }
  at::Tensor& ws = it->second;
  if (!ws.defined() || (size_t)ws.numel() < bytes) {
    ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    ws.narrow(0, 0, (int64_t)logo_sq_workspace_counter_bytes()).zero_();
  }
  return ws;
}

std::tuple<at::Tensor, at::Tensor> sq_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                          const std::optional<at::Tensor>& q_idx,
                                          const std::optional<at::Tensor>& pos, const at::Tensor& meta,
                                          const at::Tensor& cu, int64_t lanes, double scale, int64_t window) {
  const int dtype = check_attn(q, k, v);
  const int64_t n = q.size(0), hq = q.size(1), h = k.size(1), d = q.size(2);
  // Every row of o and lse is written (sparse mode: zero for unselected
  // tokens and for lse rows past each lane's rows, by the kernel).
  auto o = at::empty_like(q);
  auto lse = at::empty({hq, n}, q.options().dtype(at::kFloat));
  auto ws = window < 0 ? split_workspace(q, k, cu, dtype, true) : at::empty({0}, q.options().dtype(at::kByte));
  ok(logo_sq_fwd(cptr(q), cptr(k), cptr(v), mptr(o), lse.data_ptr<float>(), opt_ptr<int64_t>(q_idx),
                 opt_ptr<int32_t>(pos), meta.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), n, (int)cu.numel() - 1,
                 (int)hq, (int)h, (int)d, (int)v.size(2), (int)lanes, (float)scale, (int)window, dtype,
                 ws.numel() ? ws.data_ptr() : nullptr, (size_t)ws.numel(), sp()),
     "logo_sq_fwd");
  return {o, lse};
}

// One backward phase (0 delta, 1 dq, 2 dk/dv) through its C entry point.
struct Bwd {
  const at::Tensor &q, &k, &v, &o, &lse, &dout;
  const std::optional<at::Tensor>&q_idx, &pos;
  const at::Tensor &meta, &cu;
  int64_t lanes;
  double scale;
  int64_t window;
  int call(int phase, at::Tensor* delta, at::Tensor* q_sel, at::Tensor* do_sel, at::Tensor* dq, at::Tensor* dk,
           at::Tensor* dv) const {
    const int dtype = check_attn(q, k, v);
    need(o, "o", q.scalar_type());
    need(dout, "dout", q.scalar_type());
    TORCH_CHECK(o.sizes() == q.sizes() && dout.sizes() == q.sizes(), "logo_hip: o and dout must be [N, HQ, D]");
    if (phase > 0) {
      need(*delta, "delta", at::kFloat);
      TORCH_CHECK(delta->numel() == q.size(0) * q.size(1), "logo_hip: delta must be [HQ, N]");
      if (q_idx.has_value() && !generic_path(q, dtype)) {
        need(*q_sel, "q_sel", q.scalar_type());
        need(*do_sel, "do_sel", q.scalar_type());
        TORCH_CHECK(q_sel->numel() == q.numel() && do_sel->numel() == q.numel(),
                    "logo_hip: q_sel and do_sel must be [HQ, N, D]");
      }
    }
    using F = decltype(&logo_sq_bwd);
    F fn = phase == 0 ? &logo_sq_bwd_delta : phase == 1 ? &logo_sq_bwd_dq : phase == 2 ? &logo_sq_bwd_dkv
                                                                                  : &logo_sq_bwd_dqkv;
    auto p = [](at::Tensor* t) -> void* { return t && t->numel() ? t->data_ptr() : nullptr; };
    at::Tensor ws = phase >= 1 && window < 0 ? split_workspace(q, k, cu, dtype, false)
                                             : at::empty({0}, q.options().dtype(at::kByte));
    return fn(cptr(q), cptr(k), cptr(v), cptr(o), cptr(dout), lse.data_ptr<float>(),
              static_cast<float*>(p(delta)), p(q_sel), p(do_sel), p(dq), p(dk), p(dv), opt_ptr<int64_t>(q_idx),
              opt_ptr<int32_t>(pos), meta.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), q.size(0),
              (int)cu.numel() - 1, (int)q.size(1), (int)k.size(1), (int)q.size(2), (int)v.size(2), (int)lanes,
              (float)scale, (int)window, dtype, p(&ws), (size_t)ws.numel(), sp());
  }
};

#define LOGO_BWD_SCHEMA_ARGS                                                                                 \
  const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &o, const at::Tensor &lse, \
      const at::Tensor &dout, const std::optional<at::Tensor>&q_idx, const std::optional<at::Tensor>&pos,    \
      const at::Tensor &meta, const at::Tensor &cu, int64_t lanes, double scale, int64_t window

// delta [HQ, N] fp32 (rows past Sq unwritten) and, in sparse mode on the tuned
// kernels, the compacted copies q_sel / do_sel [HQ, N, D] (empty in dense mode
// and on the generic kernels, which read q and dout in place): workspaces of
// the dq and dk/dv phases, whose rows past each head's Sq are left unwritten.
std::tuple<at::Tensor, at::Tensor, at::Tensor> sq_bwd_delta(LOGO_BWD_SCHEMA_ARGS) {
  const bool sparse = q_idx.has_value() && !generic_path(q, check_attn(q, k, v));
  auto delta = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
  auto q_sel = sparse ? at::empty({q.size(1), q.size(0), q.size(2)}, q.options()) : at::empty({0}, q.options());
  auto do_sel = sparse ? at::empty_like(q_sel) : at::empty({0}, q.options());
  Bwd b{q, k, v, o, lse, dout, q_idx, pos, meta, cu, lanes, scale, window};
  ok(b.call(0, &delta, &q_sel, &do_sel, nullptr, nullptr, nullptr), "logo_sq_bwd_delta");
  return {delta, q_sel, do_sel};
}

at::Tensor sq_bwd_dq(LOGO_BWD_SCHEMA_ARGS, const at::Tensor& delta, const at::Tensor& q_sel,
                     const at::Tensor& do_sel) {
  check_attn(q, k, v);
  auto dq = at::empty_like(q);  // every row written (sparse: unselected rows zero)
  Bwd b{q, k, v, o, lse, dout, q_idx, pos, meta, cu, lanes, scale, window};
  auto dl = delta, qs = q_sel, ds = do_sel;
  ok(b.call(1, &dl, &qs, &ds, &dq, nullptr, nullptr), "logo_sq_bwd_dq");
  return dq;
}

std::tuple<at::Tensor, at::Tensor> sq_bwd_dkv(LOGO_BWD_SCHEMA_ARGS, const at::Tensor& delta,
                                              const at::Tensor& q_sel, const at::Tensor& do_sel) {
  check_attn(q, k, v);
  auto dk = at::empty_like(k);
  auto dv = at::empty_like(v);
  Bwd b{q, k, v, o, lse, dout, q_idx, pos, meta, cu, lanes, scale, window};
  auto dl = delta, qs = q_sel, ds = do_sel;
  ok(b.call(2, &dl, &qs, &ds, nullptr, &dk, &dv), "logo_sq_bwd_dkv");
  return {dk, dv};
}

// dq, dk and dv after the delta phase (one fused pass for the sliding window).
std::tuple<at::Tensor, at::Tensor, at::Tensor> sq_bwd_dqkv(LOGO_BWD_SCHEMA_ARGS, const at::Tensor& delta,
                                                           const at::Tensor& q_sel, const at::Tensor& do_sel) {
  check_attn(q, k, v);
  auto dq = at::empty_like(q);
  auto dk = at::empty_like(k);
  auto dv = at::empty_like(v);
  Bwd b{q, k, v, o, lse, dout, q_idx, pos, meta, cu, lanes, scale, window};
  auto dl = delta, qs = q_sel, ds = do_sel;
  ok(b.call(3, &dl, &qs, &ds, &dq, &dk, &dv), "logo_sq_bwd_dqkv");
  return {dq, dk, dv};
}

// The whole backward: (dq, dk, dv), its workspaces internal.
std::tuple<at::Tensor, at::Tensor, at::Tensor> sq_bwd(LOGO_BWD_SCHEMA_ARGS) {
  auto ws = sq_bwd_delta(q, k, v, o, lse, dout, q_idx, pos, meta, cu, lanes, scale, window);
  return sq_bwd_dqkv(q, k, v, o, lse, dout, q_idx, pos, meta, cu, lanes, scale, window, std::get<0>(ws),
                     std::get<1>(ws), std::get<2>(ws));
}

int thres_code(const at::Tensor& thres) {
  TORCH_CHECK(thres.numel() == 1 && (thres.scalar_type() == at::kBFloat16 || thres.scalar_type() == at::kFloat),
              "logo_hip: the threshold is one bf16 or fp32 value");
  return thres.scalar_type() == at::kBFloat16 ? LOGO_DTYPE_BF16 : LOGO_DTYPE_F32;
}

// L, G [n, H, D] bf16, gate [n] bf16 (post-sigmoid), w_l / w_g [D] -> out [n, H * D]
at::Tensor epilogue_fwd(const at::Tensor& L, const at::Tensor& G, const at::Tensor& gate, const at::Tensor& thres,
                        const at::Tensor& w_l, const at::Tensor& w_g, double eps) {
  need(L, "L", at::kBFloat16);
  need(G, "G", at::kBFloat16);
  need(gate, "gate", at::kBFloat16);
  TORCH_CHECK(L.dim() == 3 && G.sizes() == L.sizes() && gate.numel() == L.size(0), "logo_hip: epilogue shapes");
  auto out = at::empty({L.size(0), L.size(1) * L.size(2)}, L.options());
  ok(logo_epilogue_fwd(cptr(L), cptr(G), cptr(gate), cptr(thres), thres_code(thres), cptr(w_l), cptr(w_g),
                       mptr(out), L.size(0), (int)L.size(1), (int)L.size(2), (float)eps, LOGO_DTYPE_BF16, sp()),
     "logo_epilogue_fwd");
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> epilogue_bwd(
    const at::Tensor& L, const at::Tensor& G, const at::Tensor& gate, const at::Tensor& thres, const at::Tensor& w_l,
    const at::Tensor& w_g, const at::Tensor& dout, double eps) {
  need(L, "L", at::kBFloat16);
  need(dout, "dout", at::kBFloat16);
  const int64_t n = L.size(0), H = L.size(1), D = L.size(2);
  auto dL = at::empty_like(L), dG = at::empty_like(G), dgate = at::empty_like(gate);
  auto dwl = at::empty_like(w_l), dwg = at::empty_like(w_g);
  auto ws = at::empty({(int64_t)logo_epilogue_bwd_workspace_bytes(n, (int)H, (int)D)}, L.options().dtype(at::kByte));
  ok(logo_epilogue_bwd(cptr(L), cptr(G), cptr(gate), cptr(thres), thres_code(thres), cptr(w_l), cptr(w_g),
                       cptr(dout), mptr(dL), mptr(dG), mptr(dgate), mptr(dwl), mptr(dwg), n, (int)H, (int)D,
                       (float)eps, ws.data_ptr(), LOGO_DTYPE_BF16, sp()),
     "logo_epilogue_bwd");
  return {dL, dG, dgate, dwl, dwg};
}

// q [B, HQ, D], caches [B, H, T_cap, D], lens i32 [B]; gate [B] with thres, or neither.
at::Tensor decode_attn(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                       const at::Tensor& lens, const std::optional<at::Tensor>& gate,
                       const std::optional<at::Tensor>& thres, int64_t max_len, double scale) {
  need(q, "q", at::kBFloat16);
  need(lens, "lens", at::kInt);
  TORCH_CHECK(gate.has_value() == thres.has_value(), "logo_hip: gate and thres go together");
  const int64_t B = q.size(0), HQ = q.size(1), D = q.size(2);
  auto out = at::empty_like(q);
  auto ws = at::empty({(int64_t)logo_decode_workspace_bytes((int)B, (int)HQ, (int)D, (int)max_len)},
                      q.options().dtype(at::kByte));
  ok(logo_decode_attn(cptr(q), cptr(k_cache), cptr(v_cache), lens.data_ptr<int32_t>(),
                      gate.has_value() ? cptr(*gate) : nullptr, thres.has_value() ? cptr(*thres) : nullptr,
                      thres.has_value() ? thres_code(*thres) : LOGO_DTYPE_F32, mptr(out), ws.data_ptr(), (int)B,
                      (int)HQ, (int)k_cache.size(1), (int)D, k_cache.size(2), (int)max_len, (float)scale,
                      LOGO_DTYPE_BF16, sp()),
     "logo_decode_attn");
  return out;
}

// The paged cache's operators and the rotary embedding check everything themselves
// (ValueError for what they refuse), for tensors of any device, so that their Python
// callers only fill in defaults.

#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

// All tensors on one ROCm GPU.
void on_gpu(const char* what, std::initializer_list<const at::Tensor*> ts) {
  const at::Tensor* first = nullptr;
  for (const at::Tensor* t : ts) {
    if (t == nullptr) continue;
    TORCH_CHECK(t->is_cuda(), "logo_amd ops run only on a ROCm GPU (got a tensor on ", t->device(),
                "); there is no CPU fallback");
    if (first == nullptr) first = t;
    NEED(t->device() == first->device(), what, ": tensors on different devices");
  }
}
const at::Tensor* optional_ptr(const std::optional<at::Tensor>& t) { return t.has_value() ? &*t : nullptr; }

int float_code(at::ScalarType t) {
  return t == at::kBFloat16 ? LOGO_DTYPE_BF16 : t == at::kHalf ? LOGO_DTYPE_F16 : t == at::kFloat ? LOGO_DTYPE_F32 : -1;
}

// Stride of dimension d, 0 where its size makes it meaningless.
int64_t stride_of(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// Whether no two rows (last dimension) of x share memory: from the smallest stride up,
// each dimension steps over what the ones before it span.
bool rows_apart(const at::Tensor& x) {
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t d = 0; d < x.dim() - 1; ++d)
    if (x.size(d) > 1) dims.emplace_back(x.stride(d), x.size(d));
  std::sort(dims.begin(), dims.end());
  int64_t extent = x.size(-1);
  for (const auto& [st, n] : dims) {
    if (st < extent) return false;
    extent += st * (n - 1);
  }
  return true;
}

// Whether the stretches of memory that x and y lie in overlap.
bool overlap(const at::Tensor& x, const at::Tensor& y) {
  if (x.numel() == 0 || y.numel() == 0) return false;
  auto end = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return static_cast<const char*>(t.data_ptr()) + (last + 1) * t.element_size();
  };
  return static_cast<const char*>(x.data_ptr()) < end(y) && static_cast<const char*>(y.data_ptr()) < end(x);
}

// What was written in place is another version to autograd.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Shapes and types of a paged cache and a call's sequences.
void check_cache(const char* what, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
                 const at::Tensor& cu, const at::Tensor& lens) {
  NEED(k_pages.dim() == 4 && v_pages.sizes() == k_pages.sizes() && v_pages.scalar_type() == k_pages.scalar_type(), what,
       ": k_pages and v_pages must be [P, H, page_size, D] of one shape and type");
  const int code = float_code(k_pages.scalar_type());
  NEED(code == LOGO_DTYPE_BF16 || code == LOGO_DTYPE_F16, what, " takes bf16 or fp16 pages, got ", k_pages.scalar_type());
  NEED(table.dim() == 2 && cu.dim() == 1 && lens.dim() == 1, what,
       ": block_table must be [S, M], cu_seqlens [S + 1], lens [S]");
  for (const at::Tensor* t : {&table, &cu, &lens})
    NEED(t->scalar_type() == at::kInt, what, ": block_table, cu_seqlens and lens must be int32");
  const int64_t S = lens.size(0), page = k_pages.size(2), D = k_pages.size(3);
  NEED(table.size(0) == S && cu.size(0) == S + 1, what, ": block_table and cu_seqlens do not match ", S, " sequences");
  NEED(D == 64 || D == 128, what, ": head dim ", D, " unsupported (64 or 128)");
  NEED(page >= 16 && page <= 65536 && (page & (page - 1)) == 0, what,
       ": page_size must be a power of two in [16, 65536], got ", page);
  for (const at::Tensor* t : {&k_pages, &v_pages})
    NEED(t->stride(3) == 1 && stride_of(*t, 0) % 8 == 0 && stride_of(*t, 1) % 8 == 0 && t->stride(2) % 8 == 0 &&
             t->stride(2) >= D && aligned16(*t),
         what, ": rows of the pages must be dense and 16-byte aligned");
}

logo_paged_cache cache_arg(const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
                           const at::Tensor& cu, const at::Tensor& lens) {
  logo_paged_cache c{};
  c.k = k_pages.data_ptr();
  c.v = v_pages.data_ptr();
  c.k_page = stride_of(k_pages, 0), c.k_head = stride_of(k_pages, 1), c.k_slot = k_pages.stride(2);
  c.v_page = stride_of(v_pages, 0), c.v_head = stride_of(v_pages, 1), c.v_slot = v_pages.stride(2);
  c.pages = k_pages.size(0);
  c.heads = (int32_t)k_pages.size(1);
  c.page_size = (int32_t)k_pages.size(2);
  c.table = static_cast<const int32_t*>(table.data_ptr());
  c.table_width = (int32_t)table.size(1);
  c.table_row = table.size(0) > 1 ? table.stride(0) : table.size(1);
  c.cu = static_cast<const int32_t*>(cu.data_ptr());
  c.lens = static_cast<const int32_t*>(lens.data_ptr());
  c.nseq = (int32_t)lens.size(0);
  return c;
}

// The block table with dense rows, one behind the other.
at::Tensor dense_table(const at::Tensor& t) {
  return (t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)) ? t.contiguous() : t;
}

// x [N, H, D] with rows that 16-byte accesses reach (a copy where they do not).
at::Tensor rows16(const at::Tensor& x) {
  const bool fits = x.stride(2) == 1 && stride_of(x, 0) % 8 == 0 && stride_of(x, 1) % 8 == 0 && aligned16(x);
  return fits ? x : x.clone(at::MemoryFormat::Contiguous);
}

// out: written in place, its rows behind the last sequence left as they are; else a new
// tensor with zeros there.
at::Tensor paged_attn_impl(const at::Tensor& q_in, const at::Tensor& k_pages, const at::Tensor& v_pages,
                           const at::Tensor& table_in, const at::Tensor& cu_in, const at::Tensor& lens_in,
                           const std::optional<at::Tensor>& selection, int64_t max_q, int64_t max_len, double scale,
                           int64_t window, const std::optional<at::Tensor>& out_in) {
  const char* what = "paged_attn";
  check_cache(what, k_pages, v_pages, table_in, cu_in, lens_in);
  NEED(q_in.dim() == 3 && q_in.scalar_type() == k_pages.scalar_type() && q_in.size(2) == k_pages.size(3), what,
       ": q must be [N, HQ, D] of the pages' head dim and type");
  const int64_t N = q_in.size(0), HQ = q_in.size(1), D = q_in.size(2), H = k_pages.size(1);
  NEED(H > 0 && HQ % H == 0, what, ": ", HQ, " query heads are no multiple of the pages' ", H);
  NEED(scale > 0 && scale < std::numeric_limits<float>::max(), what, ": scale must be positive and finite, got ", scale);
  NEED(window >= -1, what, ": window must be None or >= 0, got ", window);
  NEED(!selection.has_value() || (selection->scalar_type() == at::kBool && selection->dim() == 1 && selection->size(0) == N),
       what, ": selection must be bool [N]");
  NEED(!out_in.has_value() || (out_in->sizes() == q_in.sizes() && out_in->scalar_type() == q_in.scalar_type() &&
                               out_in->is_contiguous() && aligned16(*out_in)),
       what, ": out must be contiguous, of q's shape and type");
  if (out_in.has_value()) {
    // q itself is fine: each row is read before its result is written, by the workgroups that need it
    const bool same = out_in->data_ptr() == q_in.data_ptr() && q_in.is_contiguous();
    NEED((same || !overlap(*out_in, q_in)) && !overlap(*out_in, k_pages) && !overlap(*out_in, v_pages), what,
         ": out overlaps an input");
  }
  on_gpu(what, {&k_pages, &v_pages, &table_in, &cu_in, &lens_in, &q_in, optional_ptr(selection), optional_ptr(out_in)});
  const c10::OptionalDeviceGuard guard(k_pages.device());
  if (out_in.has_value()) written(*out_in);
  at::Tensor out = out_in.has_value() ? *out_in : at::empty({N, HQ, D}, q_in.options());
  if (N == 0 || HQ == 0) return out;
  const at::Tensor q = rows16(q_in), table = dense_table(table_in), cu = cu_in.contiguous(), lens = lens_in.contiguous();
  const at::Tensor sel = selection.has_value() ? selection->contiguous() : at::Tensor();
  const logo_paged_cache c = cache_arg(k_pages, v_pages, table, cu, lens);
  const int64_t reach = (int64_t)c.table_width * c.page_size;
  const int mq = (int)(max_q < 0 ? N : std::min(max_q, N)), ml = (int)(max_len < 0 ? reach : std::min(max_len, reach));
  const int w = (int)std::min<int64_t>(window, INT32_MAX);
  const size_t bytes = logo_paged_attn_workspace_bytes(c.nseq, (int)H, (int)HQ, N, (int)D, mq, ml, w, sel.defined());
  const at::Tensor ws = bytes > 0 ? at::empty({(int64_t)bytes}, q.options().dtype(at::kByte)) : at::Tensor();
  ok(logo_paged_attn(&c, cptr(q), stride_of(q, 0), stride_of(q, 1), out.data_ptr(),
                     sel.defined() ? static_cast<const uint8_t*>(sel.data_ptr()) : nullptr, (int)HQ, N, (int)D, mq, ml,
                     (float)scale, w, !out_in.has_value(), ws.defined() ? ws.data_ptr() : nullptr, bytes,
                     float_code(q.scalar_type()), sp()),
     "logo_paged_attn");
  return out;
}
at::Tensor paged_attn(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
                      const at::Tensor& cu, const at::Tensor& lens, const std::optional<at::Tensor>& selection,
                      int64_t max_q, int64_t max_len, double scale, int64_t window) {
  return paged_attn_impl(q, k_pages, v_pages, table, cu, lens, selection, max_q, max_len, scale, window, std::nullopt);
}
void paged_attn_out(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
                    const at::Tensor& cu, const at::Tensor& lens, const std::optional<at::Tensor>& selection,
                    int64_t max_q, int64_t max_len, double scale, int64_t window, const at::Tensor& out) {
  paged_attn_impl(q, k_pages, v_pages, table, cu, lens, selection, max_q, max_len, scale, window, out);
}

// How heads are rotated: checks, and the turns' pointer.
const uint64_t* check_plan(const char* what, int64_t D, const at::Tensor& turns, int64_t head_dim, int64_t rot) {
  NEED(head_dim == D, what, ": the plan is for head dim ", head_dim, ", not ", D);
  NEED(rot >= 0 && rot <= D && rot % 2 == 0 && turns.scalar_type() == at::kLong && turns.dim() == 1 &&
           turns.size(0) == rot / 2 && turns.is_contiguous(),
       what, ": the plan's turns must be int64 [rot_dim / 2]");
  return static_cast<const uint64_t*>(turns.data_ptr());
}

// Rotated q [N, HQ, D] (an empty tensor without q); turns: none, keys are stored as they are.
at::Tensor paged_append(const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& k_pages,
                        const at::Tensor& v_pages, const at::Tensor& table_in, const at::Tensor& cu_in,
                        const at::Tensor& lens_in, const std::optional<at::Tensor>& q_in,
                        const std::optional<at::Tensor>& turns, int64_t head_dim, int64_t rot, bool interleaved,
                        double amplitude) {
  const char* what = "paged_append";
  check_cache(what, k_pages, v_pages, table_in, cu_in, lens_in);
  NEED(k_in.dim() == 3 && v_in.sizes() == k_in.sizes() && k_in.scalar_type() == k_pages.scalar_type() &&
           v_in.scalar_type() == k_in.scalar_type() && k_in.size(1) == k_pages.size(1) && k_in.size(2) == k_pages.size(3),
       what, ": k and v must be [N, H, D] of the pages' heads, head dim and type");
  const int64_t N = k_in.size(0), D = k_in.size(2);
  NEED(!q_in.has_value() || (q_in->dim() == 3 && q_in->size(0) == N && q_in->size(2) == D &&
                             q_in->scalar_type() == k_in.scalar_type()),
       what, ": q must be [N, HQ, D] of k's type");
  const uint64_t* tp = turns.has_value() ? check_plan(what, D, *turns, head_dim, rot) : nullptr;
  NEED(rows_apart(k_pages) && rows_apart(v_pages) && (k_pages.numel() == 0 || k_pages.data_ptr() != v_pages.data_ptr()),
       what, ": rows of the pages share memory");
  on_gpu(what, {&k_pages, &v_pages, &table_in, &cu_in, &lens_in, &k_in, &v_in, optional_ptr(q_in), optional_ptr(turns)});
  const c10::OptionalDeviceGuard guard(k_pages.device());
  written(k_pages);
  written(v_pages);
  const int64_t HQ = q_in.has_value() ? q_in->size(1) : 0;
  at::Tensor out = at::empty({q_in.has_value() ? N : 0, HQ, D}, k_in.options());
  if (N == 0 || k_in.size(1) == 0) return out;
  const at::Tensor k = rows16(k_in), v = rows16(v_in), q = HQ > 0 ? rows16(*q_in) : at::Tensor();
  const at::Tensor table = dense_table(table_in), cu = cu_in.contiguous(), lens = lens_in.contiguous();
  if (lens.size(0) == 0) return out.zero_();
  const logo_paged_cache c = cache_arg(k_pages, v_pages, table, cu, lens);
  ok(logo_paged_append(&c, cptr(k), stride_of(k, 0), stride_of(k, 1), cptr(v), stride_of(v, 0), stride_of(v, 1),
                       q.defined() ? cptr(q) : nullptr, q.defined() ? stride_of(q, 0) : 0,
                       q.defined() ? stride_of(q, 1) : 0, q.defined() ? out.data_ptr() : nullptr, (int)HQ, N, (int)D, tp,
                       tp != nullptr ? (int)rot : 0, interleaved, (float)amplitude, float_code(k.scalar_type()), sp()),
     "logo_paged_append");
  return out;
}

void check_rotary(const char* what, at::TensorList xs, const at::Tensor& pos, const at::Tensor& turns, int64_t head_dim,
                  int64_t rot) {
  NEED(xs.size() >= 1 && xs.size() <= 4, what, " takes one to four tensors");
  const at::Tensor& x0 = xs[0];
  for (const at::Tensor& x : xs) {
    bool same = x.dim() >= 3 && x.dim() == x0.dim() && x.size(-1) == head_dim && x.scalar_type() == x0.scalar_type();
    for (int64_t d = 0; same && d < x.dim() - 2; ++d) same = x.size(d) == x0.size(d);
    NEED(same, what, " needs [..., T, H, D] tensors of one type and shape prefix, D = ", head_dim);
  }
  NEED(float_code(x0.scalar_type()) >= 0, what, " takes bf16, fp16 or fp32 tensors, got ", x0.scalar_type());
  NEED(pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong, what, ": positions must be int32 or int64");
  const int64_t lead = x0.dim() - 2;
  bool fits = pos.dim() <= lead;
  for (int64_t d = 1; fits && d <= pos.dim(); ++d) fits = pos.size(-d) == 1 || pos.size(-d) == x0.size(lead - d);
  NEED(fits, what, ": positions ", pos.sizes(), " do not match the tokens ", x0.sizes().slice(0, lead));
  check_plan(what, head_dim, turns, head_dim, rot);
  for (const at::Tensor& x : xs) on_gpu(what, {&x, &pos, &turns, &x0});
}

// x [..., T, H, D] with dense rows and at most one batch dimension (a copy where it has none).
at::Tensor rows4(const at::Tensor& x) {
  const at::Tensor y = x.dim() > 4 ? x.reshape({-1, x.size(-3), x.size(-2), x.size(-1)}) : x;
  return y.size(-1) > 1 && y.stride(-1) != 1 ? y.contiguous() : y;
}

void launch_rotary(const std::vector<at::Tensor>& xs, const std::vector<at::Tensor>& ys, at::IntArrayRef lead,
                   const at::Tensor& positions, const at::Tensor& turns, int64_t rot, bool interleaved, double amplitude,
                   bool inverse) {
  logo_rows rows[4] = {};
  int live = 0;
  for (size_t i = 0; i < xs.size(); ++i) {
    const at::Tensor &x = xs[i], &y = ys[i];
    if (x.numel() == 0) continue;
    logo_rows& r = rows[live++];
    const bool batch = x.dim() == 4;
    r.x = x.data_ptr();
    r.y = y.data_ptr();
    r.x_batch = batch ? stride_of(x, 0) : 0, r.y_batch = batch ? stride_of(y, 0) : 0;
    r.x_token = stride_of(x, -3), r.y_token = stride_of(y, -3);
    r.x_head = stride_of(x, -2), r.y_head = stride_of(y, -2);
    r.heads = (int32_t)x.size(-2);
  }
  if (live == 0) return;
  const at::Tensor pos = positions.expand(lead).contiguous();
  ok(logo_rotary(rows, live, cptr(pos), pos.scalar_type() == at::kInt ? 32 : 64, pos.numel(), lead.back(),
                 (int)xs[0].size(-1), static_cast<const uint64_t*>(turns.data_ptr()), (int)rot, interleaved,
                 (float)amplitude, inverse, float_code(xs[0].scalar_type()), sp()),
     "logo_rotary");
}

std::vector<at::Tensor> rotary(at::TensorList xs, const at::Tensor& positions, const at::Tensor& turns, int64_t head_dim,
                               int64_t rot, bool interleaved, double amplitude, bool inverse) {
  check_rotary("rotary", xs, positions, turns, head_dim, rot);
  const c10::OptionalDeviceGuard guard(positions.device());
  std::vector<at::Tensor> in, out, flat;
  for (const at::Tensor& x : xs) {
    in.push_back(rows4(x));
    out.push_back(at::empty(x.sizes(), x.options()));
    flat.push_back(rows4(out.back()));
  }
  launch_rotary(in, flat, xs[0].sizes().slice(0, xs[0].dim() - 2), positions, turns, rot, interleaved, amplitude, inverse);
  return out;
}

// The rotation with its gradient, the transposed rotation of the gradients that arrive
// (by this operator again, so it has a gradient too).
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
variable_list call_rotary(at::TensorList xs, const at::Tensor& positions, const at::Tensor& turns, int64_t head_dim,
                          int64_t rot, bool interleaved, double amplitude, bool inverse) {
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("logo_hip::rotary", "").typed<std::vector<at::Tensor>(
      at::TensorList, const at::Tensor&, const at::Tensor&, int64_t, int64_t, bool, double, bool)>();
  return op.call(xs, positions, turns, head_dim, rot, interleaved, amplitude, inverse);
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  // (tensors inside a list would not be followed)
  using Opt = std::optional<at::Tensor>;
  static variable_list forward(AutogradContext* ctx, at::Tensor x0, Opt x1, Opt x2, Opt x3, at::Tensor positions,
                               at::Tensor turns, int64_t head_dim, int64_t rot, bool interleaved, double amplitude,
                               bool inverse) {
    std::vector<at::Tensor> xs{x0};
    for (const Opt& x : {x1, x2, x3})
      if (x.has_value()) xs.push_back(*x);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, turns});
    ctx->saved_data["dims"] = std::vector<int64_t>{head_dim, rot, interleaved, inverse};
    ctx->saved_data["amplitude"] = amplitude;
    at::AutoDispatchBelowADInplaceOrView below;
    return call_rotary(xs, positions, turns, head_dim, rot, interleaved, amplitude, inverse);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto d = ctx->saved_data["dims"].toIntVector();
    std::vector<at::Tensor> live;
    for (const at::Tensor& g : grads)
      if (g.defined()) live.push_back(g);
    if (!live.empty())
      live = call_rotary(live, saved[0], saved[1], d[0], d[1], d[2] != 0, ctx->saved_data["amplitude"].toDouble(), d[3] == 0);
    variable_list out;
    size_t k = 0;
    for (const at::Tensor& g : grads) out.push_back(g.defined() ? live[k++] : at::Tensor());
    out.resize(11);  // absent tensors, positions, turns and the five numbers have none
    return out;
  }
};

std::vector<at::Tensor> rotary_autograd(at::TensorList xs, const at::Tensor& positions, const at::Tensor& turns,
                                        int64_t head_dim, int64_t rot, bool interleaved, double amplitude, bool inverse) {
  // without a gradient to give, as without autograd
  bool need = false;
  if (at::GradMode::is_enabled())
    for (const at::Tensor& x : xs) need = need || x.requires_grad();
  if (!need) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_rotary(xs, positions, turns, head_dim, rot, interleaved, amplitude, inverse);
  }
  NEED(xs.size() >= 1 && xs.size() <= 4, "rotary takes one to four tensors");
  const auto x = [&](size_t i) { return i < xs.size() ? RotaryFunction::Opt(xs[i]) : std::nullopt; };
  return RotaryFunction::apply(xs[0], x(1), x(2), x(3), positions, turns, head_dim, rot, interleaved, amplitude, inverse);
}

void rotary_(at::TensorList xs, const at::Tensor& positions, const at::Tensor& turns, int64_t head_dim, int64_t rot,
             bool interleaved, double amplitude) {
  check_rotary("rotary_", xs, positions, turns, head_dim, rot);
  std::vector<at::Tensor> rows;
  for (const at::Tensor& x : xs) {
    NEED(x.dim() <= 4 && (x.size(-1) <= 1 || x.stride(-1) == 1), "rotary_ needs [T, H, D] or [B, T, H, D] tensors with dense rows");
    bool apart = rows_apart(x);
    for (const at::Tensor& y : rows) apart = apart && (x.numel() == 0 || x.data_ptr() != y.data_ptr());
    NEED(apart, "rotary_: rows share memory");
    rows.push_back(x);
  }
  for (const at::Tensor& x : xs) written(x);
  const c10::OptionalDeviceGuard guard(positions.device());
  launch_rotary(rows, rows, xs[0].sizes().slice(0, xs[0].dim() - 2), positions, turns, rot, interleaved, amplitude, false);
}

}  // namespace

TORCH_LIBRARY(logo_hip, m) {
  m.def("compact(Tensor selection, Tensor cu) -> (Tensor, Tensor, Tensor)");
  m.def("dense_meta(Tensor cu, int n_tokens) -> Tensor");
  m.def("sq_fwd(Tensor q, Tensor k, Tensor v, Tensor? q_idx, Tensor? pos, Tensor meta, Tensor cu, int lanes, "
        "float scale, int window) -> (Tensor, Tensor)");
  m.def("sq_bwd_delta(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor dout, Tensor? q_idx, "
        "Tensor? pos, Tensor meta, Tensor cu, int lanes, float scale, int window) -> (Tensor, Tensor, Tensor)");
  m.def("sq_bwd_dq(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor dout, Tensor? q_idx, Tensor? pos, "
        "Tensor meta, Tensor cu, int lanes, float scale, int window, Tensor delta, Tensor q_sel, Tensor do_sel) "
        "-> Tensor");
  m.def("sq_bwd_dkv(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor dout, Tensor? q_idx, "
        "Tensor? pos, Tensor meta, Tensor cu, int lanes, float scale, int window, Tensor delta, Tensor q_sel, "
        "Tensor do_sel) -> (Tensor, Tensor)");
  m.def("sq_bwd_dqkv(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor dout, Tensor? q_idx, "
        "Tensor? pos, Tensor meta, Tensor cu, int lanes, float scale, int window, Tensor delta, Tensor q_sel, "
        "Tensor do_sel) -> (Tensor, Tensor, Tensor)");
  m.def("sq_bwd(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor dout, Tensor? q_idx, Tensor? pos, "
        "Tensor meta, Tensor cu, int lanes, float scale, int window) -> (Tensor, Tensor, Tensor)");
  m.def("epilogue_fwd(Tensor L, Tensor G, Tensor gate, Tensor thres, Tensor w_l, Tensor w_g, float eps) -> Tensor");
  m.def("epilogue_bwd(Tensor L, Tensor G, Tensor gate, Tensor thres, Tensor w_l, Tensor w_g, Tensor dout, "
        "float eps) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("decode_attn(Tensor q, Tensor k_cache, Tensor v_cache, Tensor lens, Tensor? gate, Tensor? thres, "
        "int max_len, float scale) -> Tensor");
  m.def("paged_attn(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_table, Tensor cu_seqlens, Tensor lens, "
        "Tensor? selection, int max_q, int max_len, float scale, int window) -> Tensor");
  m.def("paged_attn_out(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_table, Tensor cu_seqlens, Tensor lens, "
        "Tensor? selection, int max_q, int max_len, float scale, int window, Tensor(a!) out) -> ()");
  m.def("paged_append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor block_table, "
        "Tensor cu_seqlens, Tensor lens, Tensor? q, Tensor? turns, int head_dim, int rot_dim, bool interleaved, "
        "float amplitude) -> Tensor");
  m.def("rotary(Tensor[] xs, Tensor positions, Tensor turns, int head_dim, int rot_dim, bool interleaved, "
        "float amplitude, bool inverse) -> Tensor[]");
  m.def("rotary_(Tensor(a!)[] xs, Tensor positions, Tensor turns, int head_dim, int rot_dim, bool interleaved, "
        "float amplitude) -> ()");
}

// These refuse tensors of other devices themselves.
TORCH_LIBRARY_IMPL(logo_hip, CompositeExplicitAutograd, m) {
  m.impl("paged_attn", &paged_attn);
  m.impl("paged_attn_out", &paged_attn_out);
  m.impl("paged_append", &paged_append);
  m.impl("rotary", &rotary);
  m.impl("rotary_", &rotary_);
}

TORCH_LIBRARY_IMPL(logo_hip, Autograd, m) { m.impl("rotary", &rotary_autograd); }

TORCH_LIBRARY_IMPL(logo_hip, CUDA, m) {
  m.impl("compact", &compact);
  m.impl("dense_meta", &dense_meta);
  m.impl("sq_fwd", &sq_fwd);
  m.impl("sq_bwd_delta", &sq_bwd_delta);
  m.impl("sq_bwd_dq", &sq_bwd_dq);
  m.impl("sq_bwd_dkv", &sq_bwd_dkv);
  m.impl("sq_bwd_dqkv", &sq_bwd_dqkv);
  m.impl("sq_bwd", &sq_bwd);
  m.impl("epilogue_fwd", &epilogue_fwd);
  m.impl("epilogue_bwd", &epilogue_bwd);
  m.impl("decode_attn", &decode_attn);
}
