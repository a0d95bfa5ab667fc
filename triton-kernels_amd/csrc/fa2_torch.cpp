// fa2_torch.cpp - the launch half of flash_attention_v2 / flash_attention_v1,
// decode_attention / speculative_decode_attention and paged_kv_append as a
// PyTorch-ROCm extension: after the Python wrapper has run the
// reference's assertion sequence (kernels/attention.py mirrors
// attention.py:762-834), one call here derives the sizes of the layout,
// makes rows 16-byte aligned, converts the index tensors, allocates the
// output and the workspace from torch's caching allocator, fills
// fa2_params and enqueues fa2_fwd (include/fa2.h) on torch's current HIP
// stream (likewise fa2_decode_fwd and fa2_kv_append).  It replaces a chain of
// Python steps (strides, pointer fields, a ctypes call) that cost ~11 us per
// call (prefill; decode with a workspace 15 to 18, append 14), more than small
// calls take on the GPU.  No attention arithmetic here.
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include <algorithm>

#include "fa2.h"
#include "fa2_ops.h"

namespace {

// Last dim contiguous and every row start 16-byte aligned (the kernels'
// requirement; kernels/_launch.py:rows_ok).
bool rows_ok(const at::Tensor& t) {
  if (t.numel() == 0) return true;
  const int64_t es = t.element_size();
  const auto addr = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.is_contiguous()) return addr % 16 == 0 && (t.size(-1) * es) % 16 == 0;
  if (t.stride(-1) != 1 || addr % 16) return false;
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    if ((t.stride(d) * es) % 16) return false;
  return true;
}

at::Tensor prep(const at::Tensor& t) { return rows_ok(t) ? t : t.contiguous(); }

// The element stride of dim d as the kernels take it.  torch keeps any stride on a
// dim of size one and calls the tensor contiguous all the same (one token of a
// wider row): the layout's own stride then.
int64_t stride_of(const at::Tensor& t, int64_t d) {
  if (!t.is_contiguous()) return t.stride(d);
  int64_t s = 1;
  for (int64_t i = d + 1; i < t.dim(); ++i) s *= std::max<int64_t>(t.size(i), 1);
  return s;
}

// (batch, head, row) element strides; token-major tensors (token, head).
void strides3(const at::Tensor& t, int64_t& sb, int64_t& sh, int64_t& ss) {
  if (t.dim() == 4) {
    sb = stride_of(t, 0);
    sh = stride_of(t, 1);
    ss = stride_of(t, 2);
  } else {
    sb = 0;
    sh = stride_of(t, 1);
    ss = stride_of(t, 0);
  }
}

at::Tensor index32(const at::Tensor& t, const at::Device& dev) {
  if (t.scalar_type() != at::kInt || !t.is_contiguous() || t.device() != dev)
    return t.to(dev, at::kInt).contiguous();
  return t;
}

at::Tensor table32(const at::Tensor& t, const at::Device& dev) {
  if (t.scalar_type() != at::kInt || t.stride(-1) != 1 || t.device() != dev)
    return t.to(dev, at::kInt).contiguous();
  return t;
}

int32_t dtype_code(at::ScalarType s) {
  switch (s) {
    case at::kHalf: return FA2_DTYPE_F16;
    case at::kBFloat16: return FA2_DTYPE_BF16;
    default: return FA2_DTYPE_F32;
  }
}

// layout: FA2_LAYOUT_*; mask: FA2_MASK_*; the tensors have passed the
// wrapper's asserts and dtype / head-dim checks.
at::Tensor fwd(at::Tensor q, at::Tensor k, at::Tensor v, int64_t layout, int64_t mask,
               c10::optional<at::Tensor> q_indptr, c10::optional<at::Tensor> kv_indptr,
               c10::optional<at::Tensor> k_block_table, c10::optional<at::Tensor> v_block_table,
               int64_t page_size, int64_t num_splits, int64_t max_workgroups, int64_t arith,
               int64_t kernel) {
  const at::Device dev = q.device();
  const c10::DeviceGuard guard(dev);
  fa2_params p;
  std::memset(&p, 0, sizeof(p));
  p.layout = static_cast<int32_t>(layout);
  p.dtype = dtype_code(q.scalar_type());
  p.mask = static_cast<int32_t>(mask);
  p.num_splits = static_cast<int32_t>(num_splits);
  p.max_workgroups = static_cast<int32_t>(max_workgroups);
  p.arith = static_cast<int32_t>(arith);
  p.kernel = static_cast<int32_t>(kernel);

  at::Tensor qi, kvi, kt, vt;
  if (layout == FA2_LAYOUT_DENSE) {
    p.batch = q.size(0);
    p.q_heads = q.size(1);
    p.q_len = q.size(2);
    p.head_dim = q.size(3);
    p.kv_heads = k.size(1);
    p.kv_len = k.size(2);
  } else if (layout == FA2_LAYOUT_RAGGED) {
    qi = index32(*q_indptr, dev);
    kvi = index32(*kv_indptr, dev);
    p.batch = q_indptr->numel() - 1;
    p.q_heads = q.size(1);
    p.q_len = q.size(0);
    p.head_dim = q.size(2);
    p.kv_heads = k.size(1);
    p.kv_len = k.size(0);
  } else {
    kvi = index32(*kv_indptr, dev);
    kt = table32(*k_block_table, dev);
    vt = table32(*v_block_table, dev);
    p.batch = q.size(0);
    p.q_heads = q.size(1);
    p.q_len = q.size(2);
    p.head_dim = q.size(3);
    p.kv_heads = k.size(1);
    p.kv_len = k.size(0);  // the caches' rows
    p.page_size = page_size;
    p.kv_len_max = k_block_table->size(1) * page_size;  // the reference's N (:834)
    p.k_table_stride = kt.stride(0);
    p.v_table_stride = vt.stride(0);
  }
  p.softmax_scale = static_cast<float>(std::pow(static_cast<double>(p.head_dim), -0.5));  // D ** -0.5 (:897)

  q = prep(q);
  k = prep(k);
  v = prep(v);
  at::Tensor out = at::empty_like(q);  // contiguous and aligned when q is
  if (!q.is_contiguous() && !rows_ok(out)) out = at::empty(q.sizes(), q.options());

  strides3(q, p.q_sb, p.q_sh, p.q_ss);
  strides3(k, p.k_sb, p.k_sh, p.k_ss);
  strides3(v, p.v_sb, p.v_sh, p.v_ss);
  strides3(out, p.o_sb, p.o_sh, p.o_ss);
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.o = out.data_ptr();
  if (qi.defined()) p.q_indptr = qi.data_ptr<int32_t>();
  if (kvi.defined()) p.kv_indptr = kvi.data_ptr<int32_t>();
  if (kt.defined()) {
    p.k_block_table = kt.data_ptr<int32_t>();
    p.v_block_table = vt.data_ptr<int32_t>();
  }

  size_t ws_bytes = 0;
  int rc = fa2_fwd_workspace_least(&p, &ws_bytes);
  TORCH_CHECK(rc == FA2_OK, "flash_attention_v2: ", fa2_strerror(rc), " (fa2 status ", rc, ")");
  at::Tensor ws;
  if (ws_bytes) {
    ws = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = ws_bytes;
  }
  const hipStream_t st = c10::hip::getCurrentHIPStream(dev.index()).stream();
  rc = fa2_fwd(&p, st);
  TORCH_CHECK(rc == FA2_OK, "flash_attention_v2: ", fa2_strerror(rc), " (fa2 status ", rc, ")");
  return out;
}

// Rows r = (head in group) * M + m of a kv-head group form one strided run
// (kernels/decode.py:run_ok), t [B,QH,M,D].
bool run_ok(const at::Tensor& t, int64_t M) {
  return rows_ok(t) && (M == 1 || stride_of(t, 1) == M * stride_of(t, 2));
}

// decode_attention (q [B,QH,D]) and speculative_decode_attention (q
// [B,QH,M,D]) after the Python wrapper's assertions and shape checks; null when
// the library refuses the call (the wrapper then reports it).
c10::optional<at::Tensor> decode(at::Tensor q, at::Tensor k, at::Tensor v, int64_t layout,
                                 bool causal, c10::optional<at::Tensor> kv_indptr,
                                 c10::optional<at::Tensor> k_block_table,
                                 c10::optional<at::Tensor> v_block_table, int64_t page_size,
                                 int64_t num_splits) {
  const at::Device dev = q.device();
  const c10::DeviceGuard guard(dev);
  at::Tensor out = at::empty_like(q);
  const bool squeeze = q.dim() == 3;
  at::Tensor q4 = squeeze ? q.unsqueeze(2) : q;
  at::Tensor out4 = squeeze ? out.unsqueeze(2) : out;
  const int64_t M = q4.size(2);
  if (layout == FA2_LAYOUT_PAGED && k.dim() == 4) {
    k = k.reshape({-1, k.size(2), k.size(3)});
    v = v.reshape({-1, v.size(2), v.size(3)});
  }
  k = prep(k);
  v = prep(v);
  if (!run_ok(q4, M)) q4 = q4.contiguous();
  const bool direct = run_ok(out4, M);
  at::Tensor dst = direct ? out4 : at::empty(out4.sizes(), out4.options());

  fa2_params p;
  std::memset(&p, 0, sizeof(p));
  p.layout = static_cast<int32_t>(layout);
  p.dtype = dtype_code(q4.scalar_type());
  p.mask = causal ? FA2_MASK_CAUSAL_BOTTOM_RIGHT : FA2_MASK_NONE;
  p.num_splits = static_cast<int32_t>(num_splits);
  p.batch = q4.size(0);
  p.q_heads = q4.size(1);
  p.q_len = M;
  p.head_dim = q4.size(3);
  at::Tensor kvi, kt, vt;
  if (layout == FA2_LAYOUT_DENSE) {
    p.kv_heads = k.size(1);
    p.kv_len = k.size(2);
  } else {
    p.kv_heads = k.size(1);
    p.kv_len = k.size(0);
    kvi = index32(*kv_indptr, dev);
    p.kv_indptr = kvi.data_ptr<int32_t>();
    if (layout == FA2_LAYOUT_PAGED) {
      kt = table32(*k_block_table, dev);
      vt = table32(*v_block_table, dev);
      p.page_size = page_size;
      p.kv_len_max = kt.size(1) * page_size;
      p.k_table_stride = kt.stride(0);
      p.v_table_stride = vt.stride(0);
      p.k_block_table = kt.data_ptr<int32_t>();
      p.v_block_table = vt.data_ptr<int32_t>();
    }
  }
  p.softmax_scale = static_cast<float>(std::pow(static_cast<double>(p.head_dim), -0.5));
  // M = 1: the rows of a unit are its heads, the row stride is the head stride
  auto set_strides = [&](const at::Tensor& t, int64_t& sb, int64_t& sh, int64_t& ss) {
    sb = stride_of(t, 0);
    sh = stride_of(t, 1);
    ss = stride_of(t, M > 1 ? 2 : 1);
  };
  set_strides(q4, p.q_sb, p.q_sh, p.q_ss);
  set_strides(dst, p.o_sb, p.o_sh, p.o_ss);
  strides3(k, p.k_sb, p.k_sh, p.k_ss);
  strides3(v, p.v_sb, p.v_sh, p.v_ss);
  p.q = q4.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.o = dst.data_ptr();

  size_t ws_bytes = 0;
  if (fa2_decode_workspace_size(&p, &ws_bytes) != FA2_OK) return c10::nullopt;
  at::Tensor ws;
  if (ws_bytes) {
    ws = at::empty({static_cast<int64_t>(ws_bytes)}, q4.options().dtype(at::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = ws_bytes;
  }
  const hipStream_t st = c10::hip::getCurrentHIPStream(dev.index()).stream();
  if (fa2_decode_fwd(&p, st) != FA2_OK) return c10::nullopt;
  if (!direct) out4.copy_(dst);
  return out;
}

// paged_kv_append after the Python wrapper's checks: caches [rows, H, D], new
// rows [T, H, D] with the strides K and V share.  Returns the fa2 status.
int64_t append(const at::Tensor& kc, const c10::optional<at::Tensor>& vc, const at::Tensor& k_table,
               const c10::optional<at::Tensor>& v_table, const at::Tensor& kn,
               const c10::optional<at::Tensor>& vn, const at::Tensor& new_indptr, int64_t page_size,
               const c10::optional<at::Tensor>& start_pos) {
  const at::Device dev = kc.device();
  const c10::DeviceGuard guard(dev);
  const at::Tensor ip = index32(new_indptr, dev);
  const at::Tensor kt = table32(k_table, dev);
  at::Tensor sp, vt;
  fa2_kv_append_params p;
  std::memset(&p, 0, sizeof(p));
  p.dtype = dtype_code(kc.scalar_type());
  p.batch = new_indptr.numel() - 1;
  p.kv_heads = kc.size(1);
  p.head_dim = kc.size(2);
  p.num_rows = kn.size(0);
  p.page_size = page_size;
  p.num_pages = kc.size(0) / page_size;
  p.table_width = kt.size(1);
  p.k_table_stride = kt.stride(0);
  p.new_ts = stride_of(kn, 0);
  p.new_hs = stride_of(kn, 1);
  p.cache_ts = kc.stride(0);
  p.cache_hs = kc.stride(1);
  p.k_new = kn.data_ptr();
  p.k_cache = kc.data_ptr();
  p.new_indptr = ip.data_ptr<int32_t>();
  p.k_block_table = kt.data_ptr<int32_t>();
  if (start_pos) {
    sp = index32(*start_pos, dev);
    p.start_pos = sp.data_ptr<int32_t>();
  }
  if (vc) {
    vt = table32(*v_table, dev);
    p.v_table_stride = vt.stride(0);
    p.v_new = vn->data_ptr();
    p.v_cache = vc->data_ptr();
    p.v_block_table = vt.data_ptr<int32_t>();
  }
  const hipStream_t st = c10::hip::getCurrentHIPStream(dev.index()).stream();
  return fa2_kv_append(&p, st);
}

// ---- operators around the attention (include/fa2_ops.h) ----------------------

// A small operand (weights, table) contiguous from a 16-byte boundary.
at::Tensor packed(const at::Tensor& t) {
  if (t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// Rows as the kernels take them.  (A contiguous tensor off a 16-byte boundary is
// copied too, which contiguous() would not do.)
at::Tensor ready(const at::Tensor& t) {
  return rows_ok(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

// The functions below make the checks of the Python wrappers themselves (the
// chain of attribute reads there costs 2 to 4 us per call) and return kRefused for
// arguments that do not pass: the wrapper then runs its own and raises.
constexpr int64_t kRefused = -1;

bool real_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16 || t == at::kFloat; }

// T of [T, H, D], or B * M of [B, H, M, D]
int64_t tokens_of(const at::Tensor& t) { return t.dim() == 3 ? t.size(0) : t.size(0) * t.size(2); }

bool norm_rope_ok(const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw,
                  const at::Tensor& kw, const at::Tensor& rope, const at::Tensor& positions,
                  double eps) {
  const at::Device dev = q.device();
  if (!q.is_cuda() || k.device() != dev || qw.device() != dev || kw.device() != dev ||
      rope.device() != dev || positions.device() != dev)
    return false;
  if ((q.dim() != 3 && q.dim() != 4) || (k.dim() != 3 && k.dim() != 4)) return false;
  const auto dt = q.scalar_type();
  const int64_t D = q.size(-1);
  return real_type(dt) && (D == 16 || D == 32 || D == 64 || D == 128 || D == 256) &&
         k.scalar_type() == dt && k.size(-1) == D &&
         tokens_of(k) == tokens_of(q) && qw.dim() == 1 && kw.dim() == 1 && qw.size(0) == D &&
         kw.size(0) == D && qw.scalar_type() == kw.scalar_type() &&
         (qw.scalar_type() == dt || qw.scalar_type() == at::kFloat) &&
         (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) &&
         positions.numel() == tokens_of(q) && rope.scalar_type() == at::kFloat &&
         rope.dim() == 2 && rope.size(1) <= D && rope.size(1) % 16 == 0 && eps >= 0;
}

// qk_norm_rope; (status, q, k).
std::tuple<int64_t, at::Tensor, at::Tensor> norm_rope(at::Tensor q, at::Tensor k, at::Tensor qw,
                                                      at::Tensor kw, at::Tensor rope,
                                                      at::Tensor positions, double eps,
                                                      bool interleaved) {
  if (!norm_rope_ok(q, k, qw, kw, rope, positions, eps)) return {kRefused, q, k};
  const at::Device dev = q.device();
  const c10::DeviceGuard guard(dev);
  q = ready(q);
  k = ready(k);
  qw = packed(qw);
  kw = packed(kw);
  rope = packed(rope);
  positions = positions.contiguous();
  at::Tensor qo = at::empty(q.sizes(), q.options());
  at::Tensor ko = at::empty(k.sizes(), k.options());
  fa2_norm_rope_params p;
  std::memset(&p, 0, sizeof(p));
  p.dtype = dtype_code(q.scalar_type());
  p.weight_dtype = dtype_code(qw.scalar_type());
  p.interleaved = interleaved ? 1 : 0;
  p.eps = static_cast<float>(eps);
  p.tokens = positions.numel();
  p.q_heads = q.size(1);
  p.kv_heads = k.size(1);
  p.head_dim = q.size(-1);
  p.rotary_dim = rope.size(1);
  p.positions = rope.size(0);
  p.rope_stride = rope.size(1);
  p.q_rows = q.dim() == 4 ? q.size(2) : p.tokens;
  p.k_rows = k.dim() == 4 ? k.size(2) : p.tokens;
  strides3(q, p.q_sb, p.q_sh, p.q_ss);
  strides3(k, p.k_sb, p.k_sh, p.k_ss);
  strides3(qo, p.qo_sb, p.qo_sh, p.qo_ss);
  strides3(ko, p.ko_sb, p.ko_sh, p.ko_ss);
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.q_out = qo.data_ptr();
  p.k_out = ko.data_ptr();
  p.q_weight = qw.data_ptr();
  p.k_weight = kw.data_ptr();
  p.rope = rope.data_ptr<float>();
  p.position = positions.data_ptr();
  p.position_64 = positions.scalar_type() == at::kLong ? 1 : 0;
  const hipStream_t st = c10::hip::getCurrentHIPStream(dev.index()).stream();
  return {fa2_norm_rope(&p, st), qo, ko};
}

using OptTensor = c10::optional<at::Tensor>;

// Indices of the 4-bit cache's calls.  What is outside a pool or past a table must stay
// so in 32 bits: int64 values saturate (a table entry of 2^32 is not page 0).
at::Tensor in_32_bits(const at::Tensor& t) {
  return t.scalar_type() == at::kLong ? t.clamp(INT32_MIN, INT32_MAX) : t;
}
at::Tensor fp4_index(const at::Tensor& t, const at::Device& dev) {
  return index32(in_32_bits(t), dev);
}
at::Tensor fp4_table(const at::Tensor& t, const at::Device& dev) {
  return table32(in_32_bits(t), dev);
}

// A cache's codes and scales (fp4_cache.check_cache)
bool cache_ok(const at::Tensor& c, const at::Tensor& s, const at::Device& dev) {
  if (c.device() != dev || s.device() != dev || c.scalar_type() != at::kByte ||
      s.scalar_type() != at::kByte || c.dim() != 4 || s.dim() != 4 || !c.is_contiguous() ||
      !s.is_contiguous() || c.numel() == 0)
    return false;
  const int64_t D = c.size(3) * 2;
  return (D == 64 || D == 128 || D == 256) && s.size(0) == c.size(0) && s.size(1) == c.size(1) &&
         s.size(2) == c.size(2) && s.size(3) == D / 32;
}

// The arguments that the writer and the reader share; k and v: the rows.
bool rows_args_ok(const at::Tensor& kc, const at::Tensor& ks, const OptTensor& vc,
                  const OptTensor& vs, const at::Tensor& k_table, const OptTensor& v_table,
                  const at::Tensor& k, const OptTensor& v, const at::Tensor& indptr,
                  const OptTensor& start_pos) {
  const at::Device dev = kc.device();
  if (!kc.is_cuda() || !cache_ok(kc, ks, dev) || k_table.device() != dev ||
      indptr.device() != dev || k.device() != dev)
    return false;
  const int64_t B = indptr.numel() - 1;
  if (B < 0 || k_table.dim() != 2 || k_table.size(0) < B ||
      (start_pos && start_pos->numel() < B) || !real_type(k.scalar_type()) || k.dim() != 3 ||
      k.size(1) != kc.size(1) || k.size(2) != kc.size(3) * 2)
    return false;
  if (vc.has_value() != v.has_value() || vc.has_value() != vs.has_value() ||
      vc.has_value() != v_table.has_value())
    return false;
  return !vc || (cache_ok(*vc, *vs, dev) && vc->sizes() == kc.sizes() &&
                 v_table->dim() == 2 && v_table->size(0) >= B && v->device() == dev &&
                 v->scalar_type() == k.scalar_type() && v->sizes() == k.sizes());
}

int64_t fp4_rows(bool append, const at::Tensor& kc, const at::Tensor& ks, const OptTensor& vc,
                 const OptTensor& vs, const at::Tensor& k_table, const OptTensor& v_table,
                 at::Tensor k, OptTensor v, const at::Tensor& indptr, const OptTensor& start_pos) {
  if (!rows_args_ok(kc, ks, vc, vs, k_table, v_table, k, v, indptr, start_pos)) return kRefused;
  const at::Device dev = kc.device();
  const c10::DeviceGuard guard(dev);
  if (append) {  // (the gathered tensors are contiguous and aligned)
    k = ready(k);
    if (v) v = ready(*v);
  }
  const at::Tensor ip = fp4_index(indptr, dev);
  const at::Tensor kt = fp4_table(k_table, dev);
  at::Tensor sp, vt;
  fa2_fp4_rows_params p;
  std::memset(&p, 0, sizeof(p));
  p.dtype = dtype_code(k.scalar_type());
  p.batch = indptr.numel() - 1;
  p.kv_heads = kc.size(1);
  p.head_dim = k.size(2);
  p.num_rows = k.size(0);
  p.page_size = kc.size(2);
  p.num_pages = kc.size(0);
  p.table_width = kt.size(1);
  p.k_table_stride = kt.stride(0);
  p.k_ts = stride_of(k, 0);
  p.k_hs = stride_of(k, 1);
  p.k = k.data_ptr();
  p.k_codes = kc.data_ptr<uint8_t>();
  p.k_scales = ks.data_ptr<uint8_t>();
  p.indptr = ip.data_ptr<int32_t>();
  p.k_block_table = kt.data_ptr<int32_t>();
  if (start_pos) {
    sp = fp4_index(*start_pos, dev);
    p.start_pos = sp.data_ptr<int32_t>();
  }
  if (vc) {
    vt = fp4_table(*v_table, dev);
    p.table_width = std::min(p.table_width, vt.size(1));
    p.v_table_stride = vt.stride(0);
    p.v_ts = stride_of(*v, 0);
    p.v_hs = stride_of(*v, 1);
    p.v = v->data_ptr();
    p.v_codes = vc->data_ptr<uint8_t>();
    p.v_scales = vs->data_ptr<uint8_t>();
    p.v_block_table = vt.data_ptr<int32_t>();
  }
  const hipStream_t st = c10::hip::getCurrentHIPStream(dev.index()).stream();
  return append ? fa2_fp4_append(&p, st) : fa2_fp4_gather(&p, st);
}

// paged_kv_append_fp4: writes the rows; the status.
int64_t fp4_append(const at::Tensor& kc, const at::Tensor& ks, const OptTensor& vc,
                   const OptTensor& vs, const at::Tensor& k_table, const OptTensor& v_table,
                   const at::Tensor& k, const OptTensor& v, const at::Tensor& indptr,
                   const OptTensor& start_pos) {
  return fp4_rows(true, kc, ks, vc, vs, k_table, v_table, k, v, indptr, start_pos);
}

// paged_kv_gather_fp4 into new tensors of type `like`'s; (status, k, v).
std::tuple<int64_t, at::Tensor, OptTensor> fp4_gather(
    const at::Tensor& kc, const at::Tensor& ks, const OptTensor& vc, const OptTensor& vs,
    const at::Tensor& k_table, const OptTensor& v_table, int64_t num_rows, at::ScalarType dtype,
    const at::Tensor& indptr, const OptTensor& start_pos) {
  if (num_rows < 0 || kc.dim() != 4 || !real_type(dtype)) return {kRefused, kc, vc};
  const auto opts = kc.options().dtype(dtype);
  const int64_t H = kc.size(1), D = kc.size(3) * 2;
  at::Tensor k = at::empty({num_rows, H, D}, opts);
  OptTensor v;
  if (vc) v = at::empty({num_rows, H, D}, opts);
  return {fp4_rows(false, kc, ks, vc, vs, k_table, v_table, k, v, indptr, start_pos), k, v};
}

// ... into given ones; the status.
int64_t fp4_gather_into(const at::Tensor& kc, const at::Tensor& ks, const OptTensor& vc,
                        const OptTensor& vs, const at::Tensor& k_table, const OptTensor& v_table,
                        const at::Tensor& k, const OptTensor& v, const at::Tensor& indptr,
                        const OptTensor& start_pos) {
  return fp4_rows(false, kc, ks, vc, vs, k_table, v_table, k, v, indptr, start_pos);
}

// decode_attention_fp4 (q [B,QH,D]) and speculative_decode_attention_fp4 (q
// [B,QH,M,D]): `dims` is q's; (status, output).
std::tuple<int64_t, at::Tensor> fp4_decode(const at::Tensor& q, const at::Tensor& kc,
                                           const at::Tensor& ks, const at::Tensor& vc,
                                           const at::Tensor& vs, const at::Tensor& lens,
                                           const at::Tensor& k_table, const at::Tensor& v_table,
                                           bool causal, int64_t dims) {
  const at::Device dev = q.device();
  const auto dt = q.scalar_type();
  if (!q.is_cuda() || q.dim() != dims || (dims == 4 && q.size(2) > 16) || kc.dim() != 4 ||
      (dt != at::kHalf && dt != at::kBFloat16) || !cache_ok(kc, ks, dev) ||
      !cache_ok(vc, vs, dev) || vc.sizes() != kc.sizes() || q.size(-1) != kc.size(3) * 2 ||
      q.size(1) == 0 || q.size(1) % kc.size(1) != 0 || lens.device() != dev ||
      k_table.device() != dev || v_table.device() != dev || lens.numel() < q.size(0) ||
      k_table.dim() != 2 || v_table.dim() != 2 || k_table.size(0) < q.size(0) ||
      v_table.size(0) < q.size(0))
    return {kRefused, q};
  const c10::DeviceGuard guard(dev);
  at::Tensor out = at::empty(q.sizes(), q.options());
  const bool squeeze = q.dim() == 3;
  at::Tensor q4 = squeeze ? q.unsqueeze(2) : q;
  const at::Tensor o4 = squeeze ? out.unsqueeze(2) : out;
  const int64_t M = q4.size(2);
  if (!run_ok(q4, M)) q4 = q4.clone(at::MemoryFormat::Contiguous);
  const at::Tensor li = fp4_index(lens, dev);
  const at::Tensor kt = fp4_table(k_table, dev);
  const at::Tensor vt = fp4_table(v_table, dev);
  fa2_fp4_decode_params p;
  std::memset(&p, 0, sizeof(p));
  p.dtype = dtype_code(q.scalar_type());
  p.mask = causal ? FA2_MASK_CAUSAL_BOTTOM_RIGHT : FA2_MASK_NONE;
  p.batch = q4.size(0);
  p.q_heads = q4.size(1);
  p.kv_heads = kc.size(1);
  p.head_dim = q4.size(3);
  p.q_len = M;
  p.page_size = kc.size(2);
  p.num_pages = kc.size(0);
  p.table_width = std::min(kt.size(1), vt.size(1));
  p.k_table_stride = kt.stride(0);
  p.v_table_stride = vt.stride(0);
  auto set_strides = [&](const at::Tensor& t, int64_t& sb, int64_t& sh, int64_t& ss) {
    sb = stride_of(t, 0);
    sh = stride_of(t, 1);
    ss = stride_of(t, M > 1 ? 2 : 1);
  };
  set_strides(q4, p.q_sb, p.q_sh, p.q_ss);
  set_strides(o4, p.o_sb, p.o_sh, p.o_ss);
  p.q = q4.data_ptr();
  p.o = out.data_ptr();
  p.k_codes = kc.data_ptr<uint8_t>();
  p.k_scales = ks.data_ptr<uint8_t>();
  p.v_codes = vc.data_ptr<uint8_t>();
  p.v_scales = vs.data_ptr<uint8_t>();
  p.kv_lens = li.data_ptr<int32_t>();
  p.k_block_table = kt.data_ptr<int32_t>();
  p.v_block_table = vt.data_ptr<int32_t>();
  p.softmax_scale = static_cast<float>(std::pow(static_cast<double>(p.head_dim), -0.5));
  size_t ws_bytes = 0;
  int rc = fa2_fp4_decode_workspace_size(&p, &ws_bytes);
  if (rc != FA2_OK) return {rc, out};
  at::Tensor ws;
  if (ws_bytes) {
    ws = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = ws_bytes;
  }
  const hipStream_t st = c10::hip::getCurrentHIPStream(dev.index()).stream();
  return {fa2_fp4_decode(&p, st), out};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("fwd", &fwd, "enqueue fa2_fwd for checked tensors; returns the output");
  m.def("decode", &decode, "enqueue fa2_decode_fwd for checked tensors; the output, or None");
  m.def("append", &append, "enqueue fa2_kv_append for checked tensors; the fa2 status");
  m.def("norm_rope", &norm_rope, "enqueue fa2_norm_rope; (fa2 status, -1: bad arguments, q, k)");
  m.def("fp4_append", &fp4_append, "enqueue fa2_fp4_append; the fa2 status, -1: bad arguments");
  m.def("fp4_gather", &fp4_gather, "enqueue fa2_fp4_gather; (fa2 status or -1, k, v)");
  m.def("fp4_gather_into", &fp4_gather_into, "enqueue fa2_fp4_gather; the fa2 status or -1");
  m.def("fp4_decode", &fp4_decode,
        "enqueue fa2_fp4_decode; (fa2 status or -1, output)");
}
