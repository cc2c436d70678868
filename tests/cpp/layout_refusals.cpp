// Calls one template of include/anygpu with tensors of a given layout and no memory behind them: either an ACASSERT refuses the layout (the
// message is printed, exit code 1), or the call goes on to what comes next and fails there for want of memory, before any kernel.
// Usage: layout_refusals CASE
#include <cstdio>
#include <map>
#include <functional>

#include "anygpu/fused/causal_conv1d.hpp"
#include "anygpu/fused/selective_scan.hpp"
#include "anygpu/ops/norm_ops.hpp"

template <typename dtype = float32>
static Tensor<dtype, CUDA> layout(const std::vector<int64>& shape, const std::vector<int64>& stride = {})
{
	Tensor<dtype, CUDA> t;
	t.dim = static_cast<int64>(shape.size());
	t.shape = cvt_vector2array(shape);
	t.stride = stride.empty() ? calc_default_stride(t.dim, t.shape) : cvt_vector2array(stride);
	t.mem_buffer = std::make_shared<MemoryBuffer<CUDA>>(0);
	return t;
}

typedef Tensor<float32, CUDA> T;

// batch 2, 7 tokens, 4 channels, g groups, 3 states
struct Scan
{
	T x = layout({ 2, 7, 4 }), dt = x, A = layout({ 4, 3 }), B, C, dy = x, ck = layout({ 2 * 1 * 4 * 3 });
	explicit Scan(int64 g = 2) : B(layout({ 2, 7, g, 3 })), C(B) {}
	SelectiveScanArgs<float32> args() const { return { x, dt, A, B, C }; }
	void run() const { tensor_selective_scan(args()); }
	void gradient() const { tensor_selective_scan_backward(dy, args(), ck); }
};
struct Step
{
	T state = layout({ 2, 4, 3 }), x = layout({ 2, 4 }), dt = x, A = layout({ 4, 3 }), B, C;
	explicit Step(int64 g = 2) : B(layout({ 2, g, 3 })), C(B) {}
	void run() { tensor_selective_scan_update(state, x, dt, A, B, C); }
};

// 2 x 7 rows of 5 columns
struct Norm
{
	T x = layout({ 2, 7, 5 }), dy = x, w = layout({ 5 }), b = w, mean = layout({ 14 }), rstd = mean;
	void run() const { tensor_layer_norm(x, -1, w, b, 1e-5f); }
	void gradient() const { tensor_layer_norm_backward(dy, x, w, mean, rstd); }
};

// 2 x 7 tokens of 5 channels, width 4
struct Conv
{
	T x = layout({ 2, 7, 5 }), dy = x, w = layout({ 5, 4 }), b = layout({ 5 });
	void run() const { tensor_causal_conv1d_tokens(x, w, b); }
	void gradient() const { tensor_causal_conv1d_tokens_backward(dy, x, w, b); }
};

int main(int argc, char** argv)
{
	const std::map<std::string, std::function<void()>> cases = {
		// whole rows of groups out of wider rows, and one group out of wider rows, are views that the kernels take
		{ "scan", [] { Scan().run(); } },
		{ "scan gradient", [] { Scan().gradient(); } },
		{ "scan rows of groups", [] { Scan s; s.B = layout({ 2, 7, 2, 3 }, { 7 * 20, 20, 3, 1 }); s.C = s.B; s.run(); } },
		{ "scan one group of wider rows", [] { Scan s(1); s.B = layout({ 2, 7, 1, 3 }, { 7 * 20, 20, 20, 1 }); s.C = s.B; s.run(); } },
		{ "scan channels of wider rows", [] { Scan s; s.x = layout({ 2, 7, 4 }, { 7 * 9, 9, 1 }); s.run(); } },
		{ "step", [] { Step().run(); } },
		{ "step rows of groups", [] { Step s; s.B = layout({ 2, 2, 3 }, { 20, 3, 1 }); s.C = s.B; s.run(); } },
		{ "step one group of wider rows", [] { Step s(1); s.B = layout({ 2, 1, 3 }, { 20, 20, 1 }); s.C = s.B; s.run(); } },
		// states sliced out of every group: the second group is not where the kernels look
		{ "scan B of sliced states", [] { Scan s; s.B = layout({ 2, 7, 2, 3 }, { 7 * 12, 12, 6, 1 }); s.run(); } },
		{ "scan C of sliced states", [] { Scan s; s.C = layout({ 2, 7, 2, 3 }, { 7 * 12, 12, 6, 1 }); s.run(); } },
		{ "scan gradient C of sliced states", [] { Scan s; s.C = layout({ 2, 7, 2, 3 }, { 7 * 12, 12, 6, 1 }); s.gradient(); } },
		{ "scan B states apart", [] { Scan s(1); s.B = layout({ 2, 7, 1, 3 }, { 7 * 6, 6, 6, 2 }); s.run(); } },
		{ "scan channels apart", [] { Scan s; s.x = layout({ 2, 7, 4 }, { 7 * 8, 8, 2 }); s.run(); } },
		{ "scan gradient dy channels apart", [] { Scan s; s.dy = layout({ 2, 7, 4 }, { 7 * 8, 8, 2 }); s.gradient(); } },
		{ "step B of sliced states", [] { Step s; s.B = layout({ 2, 2, 3 }, { 12, 6, 1 }); s.run(); } },
		{ "step C of sliced states", [] { Step s; s.C = layout({ 2, 2, 3 }, { 12, 6, 1 }); s.run(); } },
		{ "step channels apart", [] { Step s; s.dt = layout({ 2, 4 }, { 8, 2 }); s.run(); } },
		{ "norm", [] { Norm().run(); } },
		{ "norm gradient", [] { Norm().gradient(); } },
		{ "norm of wider rows", [] { Norm s; s.x = layout({ 2, 7, 5 }, { 7 * 9, 9, 1 }); s.run(); } },
		{ "norm of one row", [] { Norm s; s.x = layout({ 5 }); s.run(); } },
		// rows cut out of every matrix: the second matrix does not follow the first one's last row
		{ "norm of cut rows", [] { Norm s; s.x = layout({ 2, 7, 5 }, { 9 * 5, 5, 1 }); s.run(); } },
		{ "norm columns apart", [] { Norm s; s.x = layout({ 2, 7, 5 }, { 7 * 10, 10, 2 }); s.run(); } },
		{ "norm gradient of cut rows", [] { Norm s; s.x = layout({ 2, 7, 5 }, { 9 * 5, 5, 1 }); s.gradient(); } },
		{ "norm gradient of cut dy", [] { Norm s; s.dy = layout({ 2, 7, 5 }, { 9 * 5, 5, 1 }); s.gradient(); } },
		{ "conv", [] { Conv().run(); } },
		{ "conv gradient", [] { Conv().gradient(); } },
		{ "conv of wider rows", [] { Conv s; s.x = layout({ 2, 7, 5 }, { 7 * 9, 9, 1 }); s.run(); } },
		// parameters and states have no stride of their own in the C ABI: slices of wider ones are not where the kernels look
		{ "conv sliced w", [] { Conv s; s.w = layout({ 5, 4 }, { 8, 1 }); s.run(); } },
		{ "conv channels apart", [] { Conv s; s.x = layout({ 2, 7, 5 }, { 7 * 10, 10, 2 }); s.run(); } },
		{ "conv gradient sliced w", [] { Conv s; s.w = layout({ 5, 4 }, { 8, 1 }); s.gradient(); } },
		{ "conv gradient channels apart", [] { Conv s; s.dy = layout({ 2, 7, 5 }, { 7 * 10, 10, 2 }); s.gradient(); } },
		{ "scan sliced A", [] { Scan s; s.A = layout({ 4, 3 }, { 6, 1 }); s.run(); } },
		{ "scan sliced initial states", [] { Scan s; T i = layout({ 2, 4, 3 }, { 24, 6, 1 });
			tensor_selective_scan(SelectiveScanArgs<float32>{ s.x, s.dt, s.A, s.B, s.C, nullptr, nullptr, nullptr, &i }); } },
		{ "scan gradient sliced dfinal states", [] { Scan s; T f = layout({ 2, 4, 3 }, { 24, 6, 1 });
			tensor_selective_scan_backward(s.dy, s.args(), s.ck, &f); } },
		{ "step sliced A", [] { Step s; s.A = layout({ 4, 3 }, { 6, 1 }); s.run(); } },
		{ "step sliced state", [] { Step s; s.state = layout({ 2, 4, 3 }, { 24, 6, 1 }); s.run(); } },
	};
	if (argc < 2 || !cases.count(argv[1])) return 2;
	cases.at(argv[1])();
	return 0;
}
