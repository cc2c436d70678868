// Selective scan with a decay per channel and state (the form of state-space layers before the per-head scan of mamba_chunk_scan.hpp):
// x, dt, z (b,l,dim), A (dim,n), B/C (b,l,g,n), D and dt_bias (dim), initial_states (b,dim,n); A is A itself and softplus of the step sizes
// is on (b200_selective_scan has the other forms). A, D, dt_bias and all states are float32. Activations may be last-axis slice views of
// wider tensors (evenly spaced rows); of B and C that holds for whole rows of g * n elements, not for some of the states of every group.
// No counterpart in anyGPU.
#pragma once

#include "../b200_call.hpp"

template <typename dtype>
struct SelectiveScanArgs
{
	const Tensor<dtype, CUDA>& x;
	const Tensor<dtype, CUDA>& dt;
	const Tensor<float32, CUDA>& A;
	const Tensor<dtype, CUDA>& B;
	const Tensor<dtype, CUDA>& C;
	const Tensor<float32, CUDA>* D = nullptr;
	const Tensor<dtype, CUDA>* z = nullptr;
	const Tensor<float32, CUDA>* dt_bias = nullptr;
	const Tensor<float32, CUDA>* initial_states = nullptr;

	b200_selective_scan_inputs c_struct() const
	{
		ACASSERT(x.dim == 3 && dt.dim == 3 && B.dim == 4 && C.dim == 4 && A.dim == 2, "x, dt (b,l,dim), A (dim,n), B/C (b,l,g,n)");
		const int64 b = x.shape[0], l = x.shape[1], d = x.shape[2], g = B.shape[2], n = B.shape[3];
		ACASSERT(A.shape[0] == d && A.shape[1] == n && C.shape[2] == g && C.shape[3] == n, "A, B and C do not match");
		auto rows = [&](const auto& t) { return t.shape[0] == b && t.shape[1] == l && t.stride[0] == l * t.stride[1] && b200_dense(t, 2); };
		ACASSERT(rows(x) && rows(dt) && rows(B) && rows(C) && (!z || rows(*z)), "batch or length do not match, or rows are not evenly spaced and dense");
		ACASSERT(dt.shape[2] == d && (!z || (z->dim == 3 && z->shape[2] == d)), "dt or z does not match x");
		ACASSERT((!D || D->numel() == d) && (!dt_bias || dt_bias->numel() == d), "D or dt_bias does not match x");
		ACASSERT(!initial_states || initial_states->numel() == b * d * n, "initial_states does not match");
		ACASSERT(b200_dense(A, 0) && (!D || b200_dense(*D, 0)) && (!dt_bias || b200_dense(*dt_bias, 0)) && (!initial_states || b200_dense(*initial_states, 0)),
			"A, D, dt_bias and initial_states need to be dense");
		return { x.buffer(), dt.buffer(), B.buffer(), C.buffer(), z ? z->buffer() : nullptr, x.stride[1], dt.stride[1], B.stride[1], C.stride[1],
			z ? z->stride[1] : 0, A.buffer(), D ? D->buffer() : nullptr, dt_bias ? dt_bias->buffer() : nullptr,
			initial_states ? initial_states->buffer() : nullptr, 0, 1, b, l, d, g, n };
	}
};

template <typename dtype>
struct SelectiveScanResult
{
	Tensor<dtype, CUDA> y;               // (b, l, dim)
	Tensor<float32, CUDA> final_states;  // (b, dim, n)
	Tensor<float32, CUDA> checkpoints;   // what the backward call starts from (empty unless asked for)
};

template <typename dtype>
inline SelectiveScanResult<dtype> tensor_selective_scan(const SelectiveScanArgs<dtype>& args, const bool want_checkpoints = false)
{
	const b200_selective_scan_inputs in = args.c_struct();
	SelectiveScanResult<dtype> r{ Tensor<dtype, CUDA>(args.x.dim, args.x.shape),
		Tensor<float32, CUDA>(std::vector<int64>{ in.batch, in.dim, in.d_state }), Tensor<float32, CUDA>() };
	float* ck = nullptr;
	if (want_checkpoints)
	{
		const size_t bytes = b200_selective_scan_checkpoint_bytes(in.batch, in.seqlen, in.dim, in.d_state);
		r.checkpoints = Tensor<float32, CUDA>(std::vector<int64>{ static_cast<int64>(bytes / sizeof(float)) });
		ck = r.checkpoints.buffer();
	}
	const size_t ws_bytes = b200_selective_scan_workspace_bytes(in.batch, in.seqlen, in.dim, in.ngroups, in.d_state);
	void* ws = b200_workspace(ws_bytes);
	b200_check(b200_selective_scan(b200_dtype_of<dtype>(), &in, r.y.buffer(), in.dim, r.final_states.buffer(), ck, ws, ws_bytes, nullptr),
		"tensor_selective_scan");
	return r;
}

// One token: state (b,dim,n) float32 advanced IN PLACE; x, dt, z (b,dim), B/C (b,g,n) -> y (b,dim).
template <typename dtype>
inline Tensor<dtype, CUDA> tensor_selective_scan_update(Tensor<float32, CUDA>& state, const Tensor<dtype, CUDA>& x, const Tensor<dtype, CUDA>& dt,
	const Tensor<float32, CUDA>& A, const Tensor<dtype, CUDA>& B, const Tensor<dtype, CUDA>& C, const Tensor<float32, CUDA>* D = nullptr,
	const Tensor<dtype, CUDA>* z = nullptr, const Tensor<float32, CUDA>* dt_bias = nullptr)
{
	ACASSERT(x.dim == 2 && dt.dim == 2 && B.dim == 3 && C.dim == 3 && A.dim == 2, "x, dt (b,dim), A (dim,n), B/C (b,g,n)");
	const int64 b = x.shape[0], d = x.shape[1], g = B.shape[1], n = B.shape[2];
	ACASSERT(A.shape[0] == d && A.shape[1] == n && C.shape[1] == g && C.shape[2] == n && state.numel() == b * d * n, "A, B, C or state do not match");
	ACASSERT(dt.shape[0] == b && dt.shape[1] == d && B.shape[0] == b && C.shape[0] == b, "dt, B or C does not match x");
	ACASSERT((!z || (z->dim == 2 && z->shape[0] == b && z->shape[1] == d)) && (!D || D->numel() == d) && (!dt_bias || dt_bias->numel() == d),
		"z, D or dt_bias does not match x");
	ACASSERT(b200_dense(x, 1) && b200_dense(dt, 1) && b200_dense(B, 1) && b200_dense(C, 1) && (!z || b200_dense(*z, 1)), "rows are not dense");
	ACASSERT(b200_dense(state, 0) && b200_dense(A, 0) && (!D || b200_dense(*D, 0)) && (!dt_bias || b200_dense(*dt_bias, 0)),
		"state, A, D and dt_bias need to be dense");
	Tensor<dtype, CUDA> y(x.dim, x.shape);
	b200_check(b200_selective_scan_update(b200_dtype_of<dtype>(), state.buffer(), x.buffer(), x.stride[0], dt.buffer(), dt.stride[0], A.buffer(), 0,
		B.buffer(), B.stride[0], C.buffer(), C.stride[0], D ? D->buffer() : nullptr, dt_bias ? dt_bias->buffer() : nullptr, z ? z->buffer() : nullptr,
		z ? z->stride[0] : 0, y.buffer(), d, b, d, g, n, 1, nullptr), "tensor_selective_scan_update");
	return y;
}

// Gradients; those of operands that were not given stay empty.
template <typename dtype>
struct SelectiveScanGradients
{
	Tensor<dtype, CUDA> dx, ddt, dB, dC, dz;
	Tensor<float32, CUDA> dA, dD, ddt_bias, dinitial_states;
};

template <typename dtype>
inline SelectiveScanGradients<dtype> tensor_selective_scan_backward(const Tensor<dtype, CUDA>& dy, const SelectiveScanArgs<dtype>& args,
	const Tensor<float32, CUDA>& checkpoints, const Tensor<float32, CUDA>* dfinal_states = nullptr)
{
	const b200_selective_scan_inputs in = args.c_struct();
	ACASSERT(dy.dim == 3 && dy.shape[0] == in.batch && dy.shape[1] == in.seqlen && dy.shape[2] == in.dim && dy.stride[0] == in.seqlen * dy.stride[1] &&
		b200_dense(dy, 2), "dy does not match x");
	ACASSERT(static_cast<size_t>(checkpoints.numel()) * sizeof(float) == b200_selective_scan_checkpoint_bytes(in.batch, in.seqlen, in.dim, in.d_state),
		"checkpoints are not of this call");
	ACASSERT(b200_dense(checkpoints, 0) && (!dfinal_states || (dfinal_states->numel() == in.batch * in.dim * in.d_state && b200_dense(*dfinal_states, 0))),
		"dfinal_states does not match, or it or checkpoints is not dense");
	SelectiveScanGradients<dtype> r;
	r.dx = Tensor<dtype, CUDA>(args.x.dim, args.x.shape);
	r.ddt = Tensor<dtype, CUDA>(args.x.dim, args.x.shape);
	r.dB = Tensor<dtype, CUDA>(args.B.dim, args.B.shape);
	r.dC = Tensor<dtype, CUDA>(args.B.dim, args.B.shape);
	r.dA = Tensor<float32, CUDA>(args.A.dim, args.A.shape);
	if (args.z) r.dz = Tensor<dtype, CUDA>(args.x.dim, args.x.shape);
	if (args.D) r.dD = Tensor<float32, CUDA>(std::vector<int64>{ in.dim });
	if (args.dt_bias) r.ddt_bias = Tensor<float32, CUDA>(std::vector<int64>{ in.dim });
	if (args.initial_states) r.dinitial_states = Tensor<float32, CUDA>(std::vector<int64>{ in.batch, in.dim, in.d_state });
	const int64 gn = in.ngroups * in.d_state;
	const b200_selective_scan_grads gr = { r.dx.buffer(), r.ddt.buffer(), r.dB.buffer(), r.dC.buffer(), args.z ? r.dz.buffer() : nullptr, in.dim, in.dim,
		gn, gn, in.dim, r.dA.buffer(), args.D ? r.dD.buffer() : nullptr, args.dt_bias ? r.ddt_bias.buffer() : nullptr,
		args.initial_states ? r.dinitial_states.buffer() : nullptr };
	const size_t ws_bytes = b200_selective_scan_backward_workspace_bytes(in.batch, in.seqlen, in.dim, in.ngroups, in.d_state);
	void* ws = b200_workspace(ws_bytes);
	b200_check(b200_selective_scan_backward(b200_dtype_of<dtype>(), &in, checkpoints.buffer(), dy.buffer(), dy.stride[1],
		dfinal_states ? dfinal_states->buffer() : nullptr, &gr, ws, ws_bytes, nullptr), "tensor_selective_scan_backward");
	return r;
}
