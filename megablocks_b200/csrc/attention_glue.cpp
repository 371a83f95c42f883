// PyTorch-facing host code of the windowed attention: argument checks, output allocation, tensor maps.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "kernels.h"
#include "torch_ops.h"

namespace mb {

namespace {

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }
int sm_count() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

// [batch, seq, heads, dim] 16-bit tensor that the kernels read in place: rows of whole 16 bytes on 16-byte
// boundaries, and no dimension that is broadcast.
bool in_place(const at::Tensor& t) {
  if (!t.is_cuda() || t.dim() != 4 || !(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf)) return false;
  const int64_t dim = t.size(3);
  if (dim < 8 || dim > 128 || dim % 8 != 0 || t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0)
    return false;
  for (int d = 0; d < 3; ++d)
    if (t.size(d) > 1 && (t.stride(d) <= 0 || t.stride(d) % 8 != 0 || t.stride(d) >= (int64_t(1) << 38))) return false;
  return true;
}

// (dim, seq, heads, batch) map with boxes of 64 x rows, 128-byte swizzle.
CUtensorMap make_map(const at::Tensor& t, int box_rows) {
  const int order[3] = {1, 2, 0};
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(t.size(3)), 1, 1, 1};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    dims[i + 1] = static_cast<cuuint64_t>(t.size(order[i]));
    // The stride of a dimension of one is never used, but has to be valid.
    strides[i] = static_cast<cuuint64_t>(t.size(order[i]) > 1 ? t.stride(order[i]) * 2 : 256);
  }
  const cuuint32_t box[4] = {64u, static_cast<cuuint32_t>(box_rows), 1u, 1u};
  CUtensorMap map;
  const CUresult rc = encode_tensor_map(&map, t.scalar_type() == at::kBFloat16, 4, t.data_ptr(), dims, strides, box);
  TORCH_CHECK(rc == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", int(rc));
  return map;
}

attn::Params make_params(const at::Tensor& q, const at::Tensor& k, int64_t window, int64_t sinks,
                         const OptTensor& lengths, double scale) {
  TORCH_CHECK(in_place(q) && in_place(k), "window_attention expects 16-bit CUDA tensors [batch, seq, heads, dim] with "
              "aligned rows");
  TORCH_CHECK_VALUE(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3) && k.size(2) >= 1 &&
                        q.size(2) % k.size(2) == 0 && q.size(0) >= 1 && q.size(1) >= 1 && q.size(2) >= 1,
                    "window_attention: sizes do not match");
  // Tiles, heads and sequences are the dimensions of a grid (65535 of the last two; heads and sequences share one
  // in the backward pass), rows and heads numbers of 32 bits.
  TORCH_CHECK_VALUE(q.size(0) < (int64_t(1) << 16) && q.size(1) < (int64_t(1) << 22) && q.size(2) < (int64_t(1) << 16) &&
                        q.size(0) * q.size(2) < (int64_t(1) << 31),
                    "window_attention takes fewer than 65536 sequences and heads and 4194304 tokens");
  TORCH_CHECK_VALUE(window >= 1 && sinks >= 0 && float(scale) > 0 && std::isfinite(float(scale)),
                    "window_attention: bad window, sinks or scale");
  if (lengths.has_value())
    TORCH_CHECK(lengths->device() == q.device() && lengths->is_contiguous() && lengths->scalar_type() == at::kInt &&
                    lengths->dim() == 1 && lengths->size(0) == q.size(0),
                "window_attention: lengths must be int32 [batch]");
  attn::Params p{};
  p.batch = int(q.size(0));
  p.seq = int(q.size(1));
  p.heads = int(q.size(2));
  p.kv_heads = int(k.size(2));
  p.dim = int(q.size(3));
  p.window = int(std::min<int64_t>(window, p.seq));
  p.sinks = int(std::min<int64_t>(sinks, p.seq));
  p.lengths = lengths.has_value() ? lengths->data_ptr<int>() : nullptr;
  p.scale = float(scale);
  p.seq_pad = (p.seq + attn::kPadRows - 1) / attn::kPadRows * attn::kPadRows;
  p.status = device_status(q.device());
  return p;
}

void check_like(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(in_place(t) && t.device() == like.device() && t.scalar_type() == like.scalar_type() &&
                  t.sizes() == like.sizes(), "window_attention: ", name, " does not match");
}

}  // namespace

bool window_attention_in_place(const at::Tensor& t) { return in_place(t); }

namespace {

// {out} and, where they are wanted for a backward pass, the log-sum-exp [batch, heads, padded seq] and what
// the rounding of `out` left.
std::vector<at::Tensor> window_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window,
                                       int64_t sinks, const OptTensor& lengths, double scale, bool train) {
  c10::cuda::CUDAGuard guard(q.device());
  attn::Params p = make_params(q, k, window, sinks, lengths, scale);
  TORCH_CHECK(k.device() == q.device() && k.scalar_type() == q.scalar_type(), "window_attention: k does not match q");
  check_like(v, k, "v");
  at::Tensor out = at::empty({p.batch, p.seq, p.heads, p.dim}, q.options()), lse, low;
  if (train) {
    low = at::empty_like(out);
    p.out_low = low.data_ptr();
    lse = at::empty({p.batch, p.heads, p.seq_pad}, q.options().dtype(at::kFloat));
    p.neg_lse = lse.data_ptr<float>();
  }
  const CUtensorMap map_out = make_map(out, attn::kTile);
  C10_CUDA_CHECK(attn::forward(q.scalar_type() == at::kBFloat16, make_map(q, attn::kTile), make_map(k, attn::kTile),
                               make_map(v, attn::kTile), map_out, train ? make_map(low, attn::kTile) : map_out, p,
                               stream()));
  count_launches(1);
  return {out, lse, low};
}

std::vector<at::Tensor> window_backward(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k,
                                        const at::Tensor& v, const at::Tensor& out, const at::Tensor& lse,
                                        const at::Tensor& low, int64_t window, int64_t sinks, const OptTensor& lengths,
                                        double scale, bool want_q, bool want_kv) {
  c10::cuda::CUDAGuard guard(q.device());
  attn::Params p = make_params(q, k, window, sinks, lengths, scale);
  TORCH_CHECK(k.device() == q.device() && k.scalar_type() == q.scalar_type(), "window_attention: k does not match q");
  check_like(v, k, "v");
  check_like(dout, q, "the gradient");
  check_like(out, q, "the output");
  TORCH_CHECK(out.is_contiguous() && dout.is_contiguous(), "window_attention: output and gradient must be contiguous");
  TORCH_CHECK(lse.device() == q.device() && lse.is_contiguous() && lse.scalar_type() == at::kFloat &&
                  lse.numel() == int64_t(p.batch) * p.heads * p.seq_pad, "window_attention: bad log-sum-exp");
  const bool bf16 = q.scalar_type() == at::kBFloat16;
  const int rows = attn::streamed_rows(p.dim);
  // P and dS, rounded once, leave dq and dk off by 1.43 to 1.53 times what their own rounding does, at every length;
  // as two numbers each by 1.02 (512 tokens) to 1.15 (2 tokens).  Few terms scatter, though: 1 in 20 sequences is off by
  // more than 2.3 times at 2 tokens, 1.6 at 15, 1.5 at 64, 1.45 at 512; as two numbers 1.7, 1.13, 1.07 and 1.03.  The
  // price is 7 to 10 % of the backward pass while a sequence is one streamed tile (512 x 64 tokens, 12 heads of 64: 265
  // and 285 us), 14 % at 8 x 1024 and 25 % at 4096 tokens of heads of 128.  So sequences of one tile take it, by
  // their padded length: the host does not know the others.
  p.split = p.seq <= 64;
  at::Tensor dq, dk, dv, far;
  at::Tensor delta = at::empty_like(lse);
  p.neg_lse = lse.data_ptr<float>();
  p.out_low = low.data_ptr();
  p.neg_delta = delta.data_ptr<float>();
  C10_CUDA_CHECK(attn::row_sums(bf16, out.data_ptr(), dout.data_ptr(), p, stream()));
  count_launches(1);
  if (want_kv) {
    dk = at::empty({p.batch, p.seq, p.kv_heads, p.dim}, q.options());
    dv = at::empty({p.batch, p.seq, p.kv_heads, p.dim}, q.options());
    if (p.sinks > 0) {
      // Every query sees the first tokens: their tile's stream is as long as the sequence, the others' a
      // window.  It starts first; where it would still end last, what exceeds a window is split into parts of a
      // window's length (and at least 1024 rows).  An SM runs one CTA of large heads, two of small ones.  More
      // first tokens than a tile make long streams enough to fill the SMs, and the parts' workspace grows with them.
      const int usual = attn::near_tiles(0, p.window, rows);
      const int far_tiles = std::max(0, (p.seq + rows - 1) / rows - usual);
      const int64_t streams = int64_t(p.batch) * p.kv_heads * ((p.seq + attn::kTile - 1) / attn::kTile);
      const int64_t share = streams * usual / (int64_t(sm_count()) * (p.dim > 64 ? 1 : 2));
      if (p.sinks <= attn::kTile && far_tiles > 0 && usual + far_tiles > std::max<int64_t>(usual + usual / 2, share * 3 / 4)) {
        p.far_tiles = std::max({usual, 1024 / rows, (far_tiles + 63) / 64});
        p.far_splits = (far_tiles + p.far_tiles - 1) / p.far_tiles;
        p.far_first = usual;
        far = at::empty({p.far_splits + 1, p.batch, p.kv_heads, 2, p.sinks, p.dim}, lse.options());
        p.far = far.data_ptr<float>();
      }
    }
    C10_CUDA_CHECK(attn::backward_keys(bf16, make_map(k, attn::kTile), make_map(v, attn::kTile),
                                       make_map(q, rows), make_map(dout, rows),
                                       make_map(dk, attn::kTile), make_map(dv, attn::kTile), p, stream()));
    count_launches(1);
    if (p.far_splits > 0) {
      C10_CUDA_CHECK(attn::sum_far(bf16, dk.data_ptr(), dv.data_ptr(), p, stream()));
      count_launches(1);
    }
  }
  if (want_q) {
    dq = at::empty({p.batch, p.seq, p.heads, p.dim}, q.options());
    C10_CUDA_CHECK(attn::backward_queries(bf16, make_map(q, attn::kTile), make_map(dout, attn::kTile),
                                          make_map(k, rows), make_map(v, rows),
                                          make_map(dq, attn::kTile), p, stream()));
    count_launches(1);
  }
  return {dq, dk, dv};
}

struct Window : torch::autograd::Function<Window> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                            const at::Tensor& v, int64_t window, int64_t sinks, const OptTensor& lengths, double scale) {
    const auto out = window_forward(q, k, v, window, sinks, lengths, scale, true);
    ctx->save_for_backward({q, k, v, out[0], out[1], out[2], lengths.has_value() ? *lengths : at::Tensor()});
    ctx->saved_data["how"] = std::vector<int64_t>{window, sinks};
    ctx->saved_data["scale"] = scale;
    return out[0];
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(7);
    const auto s = ctx->get_saved_variables();
    const auto how = ctx->saved_data["how"].toIntVector();
    at::Tensor dout = grads[0].contiguous();
    if (reinterpret_cast<uintptr_t>(dout.data_ptr()) % 16 != 0) dout = dout.clone();
    const bool need_k = ctx->needs_input_grad(1), need_v = ctx->needs_input_grad(2);
    const auto g = window_backward(dout, s[0], s[1], s[2], s[3], s[4], s[5], how[0], how[1],
                                   s[6].defined() ? OptTensor(s[6]) : OptTensor(), ctx->saved_data["scale"].toDouble(),
                                   ctx->needs_input_grad(0), need_k || need_v);
    out[0] = g[0];
    if (need_k) out[1] = g[1];
    if (need_v) out[2] = g[2];
    return once_differentiable(out, "window_attention");
  }
};

// 64-bit lengths are clamped before they lose their upper half.
at::Tensor int32(const at::Tensor& t, int64_t most) {
  return (t.scalar_type() == at::kInt ? t : t.clamp(0, most).to(at::kInt)).contiguous();
}

}  // namespace

// Tensors that the kernels cannot read in place are copied.  Behind a C++ node: the host passes it in a few
// microseconds each way, a Python one in some 20.
at::Tensor window_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window,
                            int64_t sinks, const OptTensor& lengths, double scale) {
  auto ready = [](const at::Tensor& t) { return in_place(t) ? t : t.clone(at::MemoryFormat::Contiguous); };
  const at::Tensor qr = ready(q), kr = ready(k), vr = ready(v);
  const OptTensor dense = lengths.has_value() ? OptTensor(int32(*lengths, q.size(1))) : OptTensor();
  if (at::GradMode::is_enabled() && (qr.requires_grad() || kr.requires_grad() || vr.requires_grad()))
    return Window::apply(qr, kr, vr, window, sinks, dense, scale);
  return window_forward(qr, kr, vr, window, sinks, dense, scale, false)[0];
}

at::Tensor window_attention_decode(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                   const at::Tensor& lengths_in, int64_t window, int64_t sinks, double scale) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.is_contiguous() && reinterpret_cast<uintptr_t>(q.data_ptr()) % 4 == 0 &&
                  in_place(k) && in_place(v) && q.device() == k.device() && k.device() == v.device() &&
                  q.scalar_type() == k.scalar_type() && k.scalar_type() == v.scalar_type() && k.sizes() == v.sizes() &&
                  q.size(0) == k.size(0) && q.size(2) == k.size(3) && q.size(1) % k.size(2) == 0,
              "window_attention_decode expects 16-bit CUDA q[batch, heads, dim] and caches [batch, capacity, kv_heads, "
              "dim] with aligned rows");
  TORCH_CHECK_VALUE(k.size(1) < (int64_t(1) << 30) && q.size(0) < (int64_t(1) << 16) && q.size(1) < (int64_t(1) << 16),
                    "window_attention_decode takes fewer than 65536 sequences and heads and 2^30 tokens");
  TORCH_CHECK(lengths_in.device() == q.device() && lengths_in.dim() == 1 && lengths_in.size(0) == q.size(0),
              "window_attention_decode: lengths must be [batch]");
  TORCH_CHECK_VALUE(window >= 1 && sinks >= 0 && float(scale) > 0 && std::isfinite(float(scale)),
                    "window_attention_decode: bad window, sinks or scale");
  c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor lengths = int32(lengths_in, k.size(1));
  at::Tensor out = at::empty_like(q);
  if (q.size(0) == 0) return out;
  attn::DecodeParams p{};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.out = out.data_ptr();
  p.k_batch = k.stride(0), p.k_row = k.stride(1), p.k_head = k.stride(2);
  p.v_batch = v.stride(0), p.v_row = v.stride(1), p.v_head = v.stride(2);
  p.lengths = lengths.data_ptr<int>();
  p.batch = int(q.size(0));
  p.capacity = int(k.size(1));
  p.heads = int(q.size(1));
  p.kv_heads = int(k.size(2));
  p.dim = int(q.size(2));
  p.window = int(std::min<int64_t>(window, p.capacity));
  p.sinks = int(std::min<int64_t>(sinks, p.capacity));
  p.scale = float(scale);
  C10_CUDA_CHECK(attn::decode(q.scalar_type() == at::kBFloat16, p, sm_count(), stream()));
  count_launches(1);
  return out;
}

}  // namespace mb
