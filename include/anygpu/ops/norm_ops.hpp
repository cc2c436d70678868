// tensor_rms_norm for CUDA tensors, float16 and float32. Same signature as anyGPU srcs/ops/norm_ops.hpp:196-228 (whose CUDA
// overload accepts float32 only); the norm region is the last axis, which is every use on the Zamba2 path (axis = -1).
#pragma once

#include "../b200_call.hpp"

template <typename dtype>
inline Tensor<dtype, CUDA> tensor_rms_norm(const Tensor<dtype, CUDA>& xt, const int32 axis, const Tensor<dtype, CUDA> wt, const dtype eps,
	const bool zero_centered = false)
{
	const int32 dim = xt.dim;
	ACASSERT((-dim <= axis && axis < dim), "axis is out of range");
	ACASSERT((dim + axis) % dim == dim - 1, "the norm region is the last axis");
	const int64 d = xt.shape[dim - 1];
	ACASSERT(wt.shape[0] == d, "wt shape is incorrect");
	Tensor<dtype, CUDA> yt(dim, xt.shape);
	const int64 xs = dim >= 2 ? xt.stride[dim - 2] : d;
	float e;
	if constexpr (std::is_same_v<dtype, float16>) e = __half2float(eps);
	else e = static_cast<float>(eps);
	b200_check(b200_rms_norm(b200_dtype_of<dtype>(), xt.buffer(), xs, wt.buffer(), yt.buffer(), d, xt.numel() / d, d, e, zero_centered ? 1 : 0,
		nullptr), "tensor_rms_norm");
	return yt;
}

// tensor_layer_norm for CUDA tensors, float16 and float32 (anyGPU srcs/ops/norm_ops.hpp; its CUDA kernel is float32 only), over the last
// axis: (x - mean) / sqrt(var + eps) * w + b. xt may be a last-axis slice view of a wider tensor. tensor_layer_norm_with_stats also returns the
// fp32 mean and 1 / sqrt(var + eps) of every row, which the backward call needs.
template <typename dtype>
struct LayerNormResult
{
	Tensor<dtype, CUDA> y;
	Tensor<float32, CUDA> mean, rstd;  // (rows)
};

template <typename dtype>
inline LayerNormResult<dtype> tensor_layer_norm_with_stats(const Tensor<dtype, CUDA>& xt, const int32 axis, const Tensor<dtype, CUDA>& wt,
	const Tensor<dtype, CUDA>& bt, const dtype eps)
{
	const int32 dim = xt.dim;
	ACASSERT((-dim <= axis && axis < dim), "axis is out of range");
	ACASSERT((dim + axis) % dim == dim - 1, "the norm region is the last axis");
	const int64 d = xt.shape[dim - 1];
	ACASSERT(wt.shape[0] == d && bt.shape[0] == d, "wt or bt shape is incorrect");
	ACASSERT(b200_even_rows(xt, dim - 1), "the rows of xt need to be evenly spaced and dense");
	const int64 rows = xt.numel() / d, xs = dim >= 2 ? xt.stride[dim - 2] : d;
	LayerNormResult<dtype> r{ Tensor<dtype, CUDA>(dim, xt.shape), Tensor<float32, CUDA>(std::vector<int64>{ rows }),
		Tensor<float32, CUDA>(std::vector<int64>{ rows }) };
	float e;
	if constexpr (std::is_same_v<dtype, float16>) e = __half2float(eps);
	else e = static_cast<float>(eps);
	b200_check(b200_layer_norm(b200_dtype_of<dtype>(), xt.buffer(), xs, wt.buffer(), bt.buffer(), r.y.buffer(), d, r.mean.buffer(), r.rstd.buffer(),
		rows, d, e, nullptr), "tensor_layer_norm");
	return r;
}

template <typename dtype>
inline Tensor<dtype, CUDA> tensor_layer_norm(const Tensor<dtype, CUDA>& xt, const int32 axis, const Tensor<dtype, CUDA>& wt,
	const Tensor<dtype, CUDA>& bt, const dtype eps)
{
	return tensor_layer_norm_with_stats(xt, axis, wt, bt, eps).y;
}

template <typename dtype>
struct LayerNormGradients
{
	Tensor<dtype, CUDA> dx;
	Tensor<float32, CUDA> dw, db;  // (dim)
};

// Gradient for dyt, shaped like xt (no counterpart in anyGPU): dx and the sums over all rows for the weight and the bias.
template <typename dtype>
inline LayerNormGradients<dtype> tensor_layer_norm_backward(const Tensor<dtype, CUDA>& dyt, const Tensor<dtype, CUDA>& xt,
	const Tensor<dtype, CUDA>& wt, const Tensor<float32, CUDA>& mean, const Tensor<float32, CUDA>& rstd)
{
	const int64 dim = xt.dim, d = xt.shape[dim - 1], rows = xt.numel() / d;
	ACASSERT(dyt.dim == dim && dyt.numel() == xt.numel() && dyt.shape[dim - 1] == d, "dyt and xt need to have the same shape");
	ACASSERT(b200_even_rows(xt, dim - 1) && b200_even_rows(dyt, dim - 1), "the rows need to be evenly spaced and dense");
	ACASSERT(wt.shape[0] == d && mean.numel() == rows && rstd.numel() == rows, "wt, mean or rstd shape is incorrect");
	LayerNormGradients<dtype> r{ Tensor<dtype, CUDA>(dim, xt.shape), Tensor<float32, CUDA>(std::vector<int64>{ d }),
		Tensor<float32, CUDA>(std::vector<int64>{ d }) };
	const size_t ws_bytes = b200_layer_norm_backward_workspace_bytes(rows, d);
	void* ws = b200_workspace(ws_bytes);
	b200_check(b200_layer_norm_backward(b200_dtype_of<dtype>(), dyt.buffer(), dim >= 2 ? dyt.stride[dim - 2] : d, xt.buffer(),
		dim >= 2 ? xt.stride[dim - 2] : d, wt.buffer(), mean.buffer(), rstd.buffer(), r.dx.buffer(), d, r.dw.buffer(), r.db.buffer(), rows, d, ws,
		ws_bytes, nullptr), "tensor_layer_norm_backward");
	return r;
}
