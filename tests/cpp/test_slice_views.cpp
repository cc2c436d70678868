// The layer norm, token-major convolution and selective scan templates of include/anygpu on slice views of wider tensors, in float16 and
// float32, against the same calls on dense copies: the same bits (layer norm: the same to within the order of its sums). Prints "TestCase [name - CUDA]: PASSED|FAILED" per check; the exit code
// reports failure.
#include <cmath>
#include <cstdio>
#include <cstring>

#include "anygpu/fused/causal_conv1d.hpp"
#include "anygpu/fused/selective_scan.hpp"
#include "anygpu/ops/norm_ops.hpp"

static int g_failed = 0;
static void report(const std::string& name, bool ok)
{
	std::printf("TestCase [%s - CUDA]: %s\n", name.c_str(), ok ? "PASSED" : "FAILED");
	if (!ok) ++g_failed;
}
template <typename dtype>
static bool same(const Tensor<dtype, CUDA>& a, const Tensor<dtype, CUDA>& b)
{
	if (a.numel() != b.numel() || a.numel() == 0) return false;
	const auto x = a.copy_to_host(), y = b.copy_to_host();
	return std::memcmp(x.buffer(), y.buffer(), sizeof(dtype) * static_cast<size_t>(a.numel())) == 0;
}
// Two results of layer norm on one input, relative 2-norm. Rows on 16 bytes are summed four columns at a time and others one by one. With u =
// 2^-24 a sum of 20 columns is off by at most 20 u of its terms, the two orders differ by 40 u, the products around it by 4 u: the means by
// 44 u mean|x|, which for these rows (standard normal, mean|x| < 1.5 sigma) is 66 u sigma; the variances by twice that, 44 u and 4 u, and rstd
// by half of it, 90 u, relative. So x - mean over sigma moves by 156 u of its size, y (which adds b) by less than 256 u; dx carries that twice,
// in xh and in mean(q xh), with 90 u of rstd and 88 u of its two sums: 490 u, less than 512 u; dw 156 u and 18 rows.
template <typename dtype>
static bool near(const Tensor<dtype, CUDA>& a, const Tensor<dtype, CUDA>& b, const double steps)
{
	if (std::is_same_v<dtype, float16>) return same(a, b);  // 20 columns of f16 are never on 16 bytes: one order
	const auto x = a.copy_to_host(), y = b.copy_to_host();
	double d = 0, n = 0;
	for (int64 i = 0; i < a.numel(); ++i)
	{
		const double e = static_cast<double>(x.buffer()[i]) - static_cast<double>(y.buffer()[i]);
		d += e * e;
		n += static_cast<double>(y.buffer()[i]) * static_cast<double>(y.buffer()[i]);
	}
	return a.numel() == b.numel() && n > 0 && std::sqrt(d) <= steps * 0x1p-24 * std::sqrt(n);
}
// A tensor of the given shape as a slice view of rows that are `wide` elements (the last `inner` dimensions make a row), and dense.
template <typename dtype>
struct Both
{
	Tensor<dtype, CUDA> view, dense;
	Both(const std::vector<int64>& shape, const int64 inner, const int64 off, const int64 wide, const int seed, const float scale = 1.f)
	{
		int64 rows = 1, row = 1;
		const int64 dim = static_cast<int64>(shape.size());
		for (int64 i = 0; i < dim; ++i) (i < dim - inner ? rows : row) *= shape[i];
		auto host = crt_random_normal_tensor<dtype, CPU>({ rows, wide }, seed, scale);
		Tensor<dtype, CPU> cut(shape);
		for (int64 r = 0; r < rows; ++r)
			for (int64 k = 0; k < row; ++k) cut.buffer()[r * row + k] = host.buffer()[r * wide + off + k];
		dense = cut.copy_to_cuda();
		view = tensor_slice_view(host.copy_to_cuda(), off, off + row);
		view.dim = dim;
		view.shape = cvt_vector2array(shape);
		view.stride = calc_default_stride(dim, view.shape);
		for (int64 i = dim - inner - 1, step = wide; i >= 0; --i)
		{
			view.stride[i] = step;
			step *= shape[i];
		}
	}
};

template <typename dtype>
static void test_scan(const std::string& type)
{
	const int64 b = 2, l = 37, d = 12, g = 2, n = 5;
	const Both<dtype> x({ b, l, d }, 1, 3, 20, 1), dt({ b, l, d }, 1, 8, 24, 2, 0.5f), z({ b, l, d }, 1, 1, 13, 3), dy({ b, l, d }, 1, 5, 17, 4);
	const Both<dtype> B({ b, l, g, n }, 2, 2, 30, 5), C({ b, l, g, n }, 2, 16, 30, 6);
	auto A = crt_random_normal_tensor<float32, CPU>({ d, n }, 7);
	for (int64 i = 0; i < d * n; ++i) A.buffer()[i] = -0.1f - A.buffer()[i] * A.buffer()[i];
	const auto cA = A.copy_to_cuda(), cD = crt_random_normal_tensor<float32, CUDA>({ d }, 8), cb = crt_random_normal_tensor<float32, CUDA>({ d }, 9);
	const auto init = crt_random_normal_tensor<float32, CUDA>({ b, d, n }, 10);
	const SelectiveScanArgs<dtype> views{ x.view, dt.view, cA, B.view, C.view, &cD, &z.view, &cb, &init };
	const SelectiveScanArgs<dtype> dense{ x.dense, dt.dense, cA, B.dense, C.dense, &cD, &z.dense, &cb, &init };
	const auto p = tensor_selective_scan(views, true), q = tensor_selective_scan(dense, true);
	report("tensor_selective_scan " + type, same(p.y, q.y) && same(p.final_states, q.final_states));
	const auto u = tensor_selective_scan_backward(dy.view, views, p.checkpoints), v = tensor_selective_scan_backward(dy.dense, dense, q.checkpoints);
	report("tensor_selective_scan_backward " + type, same(u.dx, v.dx) && same(u.ddt, v.ddt) && same(u.dB, v.dB) && same(u.dC, v.dC) && same(u.dz, v.dz) &&
		same(u.dA, v.dA) && same(u.dD, v.dD) && same(u.ddt_bias, v.ddt_bias) && same(u.dinitial_states, v.dinitial_states));
	const Both<dtype> tx({ b, d }, 1, 3, 20, 11), tdt({ b, d }, 1, 8, 24, 12, 0.5f), tz({ b, d }, 1, 1, 13, 13);
	const Both<dtype> tB({ b, g, n }, 2, 2, 30, 14), tC({ b, g, n }, 2, 16, 30, 15);
	auto s = init.copy_to_cuda(), t = init.copy_to_cuda();
	const auto ys = tensor_selective_scan_update(s, tx.view, tdt.view, cA, tB.view, tC.view, &cD, &tz.view, &cb);
	const auto yt = tensor_selective_scan_update(t, tx.dense, tdt.dense, cA, tB.dense, tC.dense, &cD, &tz.dense, &cb);
	report("tensor_selective_scan_update " + type, same(ys, yt) && same(s, t));
}

template <typename dtype>
static void test_norm_and_conv(const std::string& type)
{
	const Both<dtype> x({ 2, 9, 20 }, 1, 3, 32, 21), dy({ 2, 9, 20 }, 1, 8, 40, 22);
	const auto w = crt_random_normal_tensor<dtype, CUDA>({ 20 }, 23), bias = crt_random_normal_tensor<dtype, CUDA>({ 20 }, 24);
	const dtype eps = static_cast<dtype>(1e-5f);
	const auto p = tensor_layer_norm_with_stats(x.view, -1, w, bias, eps), q = tensor_layer_norm_with_stats(x.dense, -1, w, bias, eps);
	report("tensor_layer_norm " + type, near(p.y, q.y, 256) && near(p.rstd, q.rstd, 256));
	const auto u = tensor_layer_norm_backward(dy.view, x.view, w, p.mean, p.rstd), v = tensor_layer_norm_backward(dy.dense, x.dense, w, q.mean, q.rstd);
	report("tensor_layer_norm_backward " + type, near(u.dx, v.dx, 512) && near(u.dw, v.dw, 512) && near(u.db, v.db, 512));
	const auto cw = crt_random_normal_tensor<dtype, CUDA>({ 20, 4 }, 25, 0.5f);
	report("tensor_causal_conv1d_tokens " + type, same(tensor_causal_conv1d_tokens(x.view, cw, bias), tensor_causal_conv1d_tokens(x.dense, cw, bias)));
	const auto g = tensor_causal_conv1d_tokens_backward(dy.view, x.view, cw, bias), h = tensor_causal_conv1d_tokens_backward(dy.dense, x.dense, cw, bias);
	report("tensor_causal_conv1d_tokens_backward " + type, same(g.dx, h.dx));
}

int main()
{
	test_scan<float16>("f16");
	test_scan<float32>("f32");
	test_norm_and_conv<float16>("f16");
	test_norm_and_conv<float32>("f32");
	return g_failed ? 1 : 0;
}
