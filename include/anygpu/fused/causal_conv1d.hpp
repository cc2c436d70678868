// tensor_causal_conv1d for CUDA tensors (float16 and float32) and the decode-step update.
// Same contract as anyGPU srcs/fused/causal_conv1d.hpp:90-117: xt (batch, dims, seq_len), wt (dims, width <= 4), bt (dims)
// -> silu(conv1d(x, w.unsqueeze(1), b, padding=width-1, groups=dims))[..., :seq_len]. The reference's CUDA overload is
// float32-only; here float16 is the main path (fp32 accumulation).
#pragma once

#include "../b200_call.hpp"

template <typename dtype>
inline Tensor<dtype, CUDA> tensor_causal_conv1d(const Tensor<dtype, CUDA>& xt, const Tensor<dtype, CUDA>& wt, const Tensor<dtype, CUDA>& bt)
{
	ACASSERT(xt.dim == 3, "xt needs to be 3 dimensional");
	ACASSERT(xt.shape[1] == wt.shape[0], "xt and wt need to have the same dims");
	ACASSERT(wt.shape[0] == bt.shape[0], "wt and bt need to have the same dims");
	ACASSERT(wt.shape[1] <= 4, "kernel width needs to be under 4");
	Tensor<dtype, CUDA> yt(xt.dim, xt.shape);
	b200_check(b200_causal_conv1d(b200_dtype_of<dtype>(), xt.buffer(), wt.buffer(), bt.buffer(), yt.buffer(), xt.shape[0], xt.shape[1],
		xt.shape[2], static_cast<int>(wt.shape[1]), nullptr), "tensor_causal_conv1d");
	return yt;
}

// One decode step. x_t (batch, dims); conv_state (batch, dims, width-1), oldest input first, advanced IN PLACE.
// Step t returns column t of tensor_causal_conv1d applied to the whole history.
template <typename dtype>
inline Tensor<dtype, CUDA> tensor_causal_conv1d_update(const Tensor<dtype, CUDA>& x_t, Tensor<dtype, CUDA>& conv_state,
	const Tensor<dtype, CUDA>& wt, const Tensor<dtype, CUDA>& bt)
{
	ACASSERT(x_t.dim == 2 && conv_state.dim == 3, "x_t is (batch, dims), conv_state is (batch, dims, width-1)");
	ACASSERT(conv_state.shape[2] == wt.shape[1] - 1, "conv_state holds width-1 inputs");
	Tensor<dtype, CUDA> y_t(x_t.dim, x_t.shape);
	b200_check(b200_causal_conv1d_update(b200_dtype_of<dtype>(), x_t.buffer(), x_t.stride[0], conv_state.buffer(), wt.buffer(), bt.buffer(),
		y_t.buffer(), y_t.stride[0], x_t.shape[0], x_t.shape[1], static_cast<int>(wt.shape[1]), nullptr), "tensor_causal_conv1d_update");
	return y_t;
}

// Token-major form: xt (batch, seq_len, dims), possibly a last-axis slice view of a wider tensor; zero left padding (states come and go
// through b200_causal_conv1d_tokens).
template <typename dtype>
inline Tensor<dtype, CUDA> tensor_causal_conv1d_tokens(const Tensor<dtype, CUDA>& xt, const Tensor<dtype, CUDA>& wt, const Tensor<dtype, CUDA>& bt)
{
	ACASSERT(xt.dim == 3 && xt.shape[2] == wt.shape[0] && wt.shape[0] == bt.shape[0], "xt (batch, seq_len, dims), wt (dims, width), bt (dims)");
	ACASSERT(b200_even_rows(xt, 2) && b200_dense(wt, 0) && b200_dense(bt, 0), "the rows of xt need to be evenly spaced and dense, wt and bt dense");
	Tensor<dtype, CUDA> yt(xt.dim, xt.shape);
	b200_check(b200_causal_conv1d_tokens(b200_dtype_of<dtype>(), xt.buffer(), xt.stride[1], wt.buffer(), bt.buffer(), yt.buffer(), yt.stride[1],
		nullptr, nullptr, xt.shape[0], xt.shape[1], xt.shape[2], static_cast<int>(wt.shape[1]), nullptr), "tensor_causal_conv1d_tokens");
	return yt;
}

template <typename dtype>
struct CausalConv1dGradients
{
	Tensor<dtype, CUDA> dx;
	Tensor<float32, CUDA> dw;  // (dims, width)
	Tensor<float32, CUDA> db;  // (dims)
};

// Gradient of the token-major form for dyt, shaped like xt (no counterpart in anyGPU).
template <typename dtype>
inline CausalConv1dGradients<dtype> tensor_causal_conv1d_tokens_backward(const Tensor<dtype, CUDA>& dyt, const Tensor<dtype, CUDA>& xt,
	const Tensor<dtype, CUDA>& wt, const Tensor<dtype, CUDA>& bt)
{
	ACASSERT(xt.dim == 3 && xt.shape[2] == wt.shape[0] && wt.shape[0] == bt.shape[0], "xt (batch, seq_len, dims), wt (dims, width), bt (dims)");
	ACASSERT(dyt.dim == 3 && dyt.shape[0] == xt.shape[0] && dyt.shape[1] == xt.shape[1] && dyt.shape[2] == xt.shape[2], "dyt and xt need to have the same shape");
	ACASSERT(b200_even_rows(xt, 2) && b200_even_rows(dyt, 2) && b200_dense(wt, 0) && b200_dense(bt, 0),
		"the rows need to be evenly spaced and dense, wt and bt dense");
	const int64 b = xt.shape[0], l = xt.shape[1], d = xt.shape[2];
	const int width = static_cast<int>(wt.shape[1]);
	CausalConv1dGradients<dtype> r{ Tensor<dtype, CUDA>(xt.dim, xt.shape), Tensor<float32, CUDA>(std::vector<int64>{ d, width }),
		Tensor<float32, CUDA>(std::vector<int64>{ d }) };
	const size_t ws_bytes = b200_causal_conv1d_tokens_backward_workspace_bytes(b, l, d, width);
	void* ws = b200_workspace(ws_bytes);
	b200_check(b200_causal_conv1d_tokens_backward(b200_dtype_of<dtype>(), dyt.buffer(), dyt.stride[1], xt.buffer(), xt.stride[1], wt.buffer(),
		bt.buffer(), nullptr, r.dx.buffer(), d, r.dw.buffer(), r.db.buffer(), nullptr, b, l, d, width, ws, ws_bytes, nullptr),
		"tensor_causal_conv1d_tokens_backward");
	return r;
}
