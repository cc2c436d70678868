// Layer norm over the last axis and its gradient (tensor_layer_norm of srcs/ops/norm_ops.hpp):
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) r w + b
//   q = dy w, xh = (x - mu) r:  dx = r (q - mean(q) - xh mean(q xh));  dw = sum_rows dy xh;  db = sum_rows dy
// Both are HBM-bound (two and three passes over the activations): a row is read once, held in registers between its statistics
// and its result, and written once (8192 x 2048 f16: 14.4 us = 4.7 TB/s; gradient of 16384 x 3584: 71 us = 5.0 TB/s).
// The variance is that of the centred values (a second pass over registers): E[x^2] - mu^2 loses everything when the rows carry a common
// offset. All sums are fp32.
#include <type_traits>

#include "column_reduce.cuh"
#include "packed.cuh"
#include "tcgen05.cuh"

namespace b200 {

// Elements of a row that a thread holds in registers: 16, and 32 in the forward kernel for many long f16 rows, which keeps enough bytes on
// their way (16384 x 4096: 50 us against 58, 16384 x 7168: 105 against 140; but 16384 x 1536 23.3 against 22.7, 64 x 4096 3.5 against 3.1).
constexpr int kLnElems = 16;
constexpr int kLnMaxThreads = 512;

// Threads that share a row of `dim` elements: the fewest of 1, 2, 3, 4, 5, 6, 8, 10, 12 and 16 warps that hold it, so that many rows are in
// flight per SM and few threads idle (powers of two only: 16384 x 2560 f16 51 us instead of 37, 16384 x 5120 131 instead of 76; seven and
// fourteen warps gain nothing). (Template arguments: with a count known only at run time a row's accesses lose their immediate
// offsets, 16384 x 2048 f16 36 us instead of 29 and its gradient twice the time.)
static int ln_threads(int64_t dim)
{
	for (int warps : { 1, 2, 3, 4, 5, 6, 8, 10, 12 })
		if (static_cast<int64_t>(warps) * 32 * kLnElems >= dim) return 32 * warps;
	return kLnMaxThreads;
}
// calls f(integral_constant<threads>); LONG: rows that need at least three warps
template <bool LONG, typename F>
static int with_ln_threads(int threads, F f)
{
	if constexpr (!LONG)
	{
		if (threads == 32) return f(std::integral_constant<int, 32>{});
		if (threads == 64) return f(std::integral_constant<int, 64>{});
	}
	switch (threads / 32)
	{
	case 3: return f(std::integral_constant<int, 96>{});
	case 4: return f(std::integral_constant<int, 128>{});
	case 5: return f(std::integral_constant<int, 160>{});
	case 6: return f(std::integral_constant<int, 192>{});
	case 8: return f(std::integral_constant<int, 256>{});
	case 10: return f(std::integral_constant<int, 320>{});
	case 12: return f(std::integral_constant<int, 384>{});
	default: return f(std::integral_constant<int, 512>{});
	}
}

// Sum over the TPR threads of a row; red holds one float per warp of the CTA for each of two alternating phases.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red)
{
	v = warp_sum(v);
	if constexpr (TPR == 32) return v;
	else
	{
		constexpr int NW = TPR / 32;
		const int wid = threadIdx.x >> 5;  // threadIdx.x runs over the row, threadIdx.y over the rows of the CTA
		float* r = red + threadIdx.y * NW;
		if ((threadIdx.x & 31) == 0) r[wid] = v;
		__syncthreads();
		float t = 0.f;
#pragma unroll
		for (int i = 0; i < NW; ++i) t += r[i];
		return t;
	}
}

// V elements per access; a row longer than TPR * ELEMS is read again for what does not fit (loops that start at `tail`).
template <typename T, int V, int ELEMS, int TPR, int ROWS>
__global__ void __launch_bounds__(TPR * ROWS) layer_norm_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ w,
	const T* __restrict__ b, T* __restrict__ y, int64_t ys, float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows,
	int dim, float eps)
{
	constexpr int C = ELEMS / V;
	__shared__ float red[2][TPR * ROWS / 32];
	const int64_t row0 = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.y;
	const bool live = row0 < rows;  // the last CTA's surplus rows repeat the last row and store nothing (the barriers need them)
	const int64_t row = live ? row0 : rows - 1;
	const T* xr = x + row * xs;
	T* yr = y + row * ys;
	const int nvec = dim / V;
	Pack<T, V> p[C];
#pragma unroll
	for (int i = 0; i < C; ++i)
	{
		const int k = threadIdx.x + i * TPR;
		if (k < nvec) p[i].load(xr + k * V);
	}
	const int tail = threadIdx.x + C * TPR;
	float v[C][V], s = 0.f;
#pragma unroll
	for (int i = 0; i < C; ++i)
	{
		if (threadIdx.x + i * TPR < nvec)
		{
			p[i].unpack(v[i]);
#pragma unroll
			for (int e = 0; e < V; ++e) s += v[i][e];
		}
	}
	for (int k = tail; k < nvec; k += TPR)
	{
		Pack<T, V> t;
		float f[V];
		t.load(xr + k * V);
		t.unpack(f);
#pragma unroll
		for (int e = 0; e < V; ++e) s += f[e];
	}
	const float inv = 1.f / static_cast<float>(dim);
	const float mu = row_sum<TPR>(s, red[0]) * inv;
	float q = 0.f;
#pragma unroll
	for (int i = 0; i < C; ++i)
	{
		if (threadIdx.x + i * TPR < nvec)
		{
#pragma unroll
			for (int e = 0; e < V; ++e)
			{
				v[i][e] -= mu;
				q += v[i][e] * v[i][e];
			}
		}
	}
	for (int k = tail; k < nvec; k += TPR)
	{
		Pack<T, V> t;
		float f[V];
		t.load(xr + k * V);
		t.unpack(f);
#pragma unroll
		for (int e = 0; e < V; ++e) q += (f[e] - mu) * (f[e] - mu);
	}
	const float r = 1.f / sqrtf(row_sum<TPR>(q, red[1]) * inv + eps);
	if (!live) return;
	if (threadIdx.x == 0)
	{
		if (mean_out) mean_out[row] = mu;
		if (rstd_out) rstd_out[row] = r;
	}
	auto put = [&](int k, const float* c /* centred */) {
		float o[V];
#pragma unroll
		for (int e = 0; e < V; ++e) o[e] = c[e] * r;
		if (w)
		{
			Pack<T, V> t;
			float f[V];
			t.load(w + k * V);
			t.unpack(f);
#pragma unroll
			for (int e = 0; e < V; ++e) o[e] *= f[e];
		}
		if (b)
		{
			Pack<T, V> t;
			float f[V];
			t.load(b + k * V);
			t.unpack(f);
#pragma unroll
			for (int e = 0; e < V; ++e) o[e] += f[e];
		}
		Pack<T, V> t;
		t.pack(o);
		t.store(yr + k * V);
	};
#pragma unroll
	for (int i = 0; i < C; ++i)
	{
		const int k = threadIdx.x + i * TPR;
		if (k < nvec) put(k, v[i]);
	}
	for (int k = tail; k < nvec; k += TPR)
	{
		Pack<T, V> t;
		float f[V];
		t.load(xr + k * V);
		t.unpack(f);
#pragma unroll
		for (int e = 0; e < V; ++e) f[e] -= mu;
		put(k, f);
	}
}

// Gradient of rows that fit the registers of a CTA (dim <= TPR * kLnElems). A CTA walks rows blockIdx.x * ROWS + threadIdx.y + i *
// gridDim.x * ROWS; a thread owns the same columns of all of them, so dw and db are sums in its registers, stored as one partial row
// per (CTA, threadIdx.y) at the end: part[p][0 .. dimp) = dw, part[p][dimp .. 2 dimp) = db. Rows without a weight gradient
// (part == nullptr) skip that.
template <typename T, int V, int TPR, int ROWS>
__global__ void __launch_bounds__(TPR * ROWS) layer_norm_backward_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x,
	int64_t xs, const T* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, int64_t dxs,
	float* __restrict__ part, int64_t rows, int dim, int64_t dimp)
{
	constexpr int C = kLnElems / V;
	__shared__ float red[2][2][TPR * ROWS / 32];
	const int nvec = dim / V;
	const float inv = 1.f / static_cast<float>(dim);
	float aw[C][V], ab[C][V];
	Pack<T, V> pw[C];
#pragma unroll
	for (int i = 0; i < C; ++i)
	{
		const int k = threadIdx.x + i * TPR;
		if (w && k < nvec) pw[i].load(w + k * V);
#pragma unroll
		for (int e = 0; e < V; ++e) aw[i][e] = ab[i][e] = 0.f;
	}
	const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
	const int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.y;
	// every row group of the CTA walks as many rows (the barriers need it): the surplus ones read the last row and count for nothing
	const int64_t walk = cdiv(rows - static_cast<int64_t>(blockIdx.x) * ROWS, step);
	Pack<T, V> px[C], pd[C];
	float nmu = 0.f, nr = 0.f;
	auto fetch = [&](int64_t row) {
		if (row >= rows) row = rows - 1;
#pragma unroll
		for (int i = 0; i < C; ++i)
		{
			const int k = threadIdx.x + i * TPR;
			if (k < nvec)
			{
				px[i].load(x + row * xs + k * V);
				pd[i].load(dy + row * dys + k * V);
			}
		}
		nmu = mean[row];
		nr = rstd[row];
	};
	if (walk > 0) fetch(first);
	for (int64_t it = 0; it < walk; ++it)
	{
		const int64_t row = first + it * step;
		const bool live = row < rows;
		const float mu = nmu, r = nr;
		float xh[C][V], q[C][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
		for (int i = 0; i < C; ++i)
		{
			if (threadIdx.x + i * TPR < nvec)
			{
				float f[V], d[V], wv[V];
				px[i].unpack(f);
				pd[i].unpack(d);
				if (w) pw[i].unpack(wv);
#pragma unroll
				for (int e = 0; e < V; ++e)
				{
					xh[i][e] = (f[e] - mu) * r;
					if (live)
					{
						aw[i][e] += d[e] * xh[i][e];
						ab[i][e] += d[e];
					}
					q[i][e] = w ? d[e] * wv[e] : d[e];
					s1 += q[i][e];
					s2 += q[i][e] * xh[i][e];
				}
			}
		}
		if (it + 1 < walk) fetch(row + step);
		// two phases alternate: the barrier of this row's sums also says that everyone has read the row before the last one's
		s1 = row_sum<TPR>(s1, red[it & 1][0]) * inv;
		s2 = row_sum<TPR>(s2, red[it & 1][1]) * inv;
		if (dx && live)
		{
#pragma unroll
			for (int i = 0; i < C; ++i)
			{
				const int k = threadIdx.x + i * TPR;
				if (k < nvec)
				{
					float o[V];
#pragma unroll
					for (int e = 0; e < V; ++e) o[e] = r * (q[i][e] - s1 - xh[i][e] * s2);
					Pack<T, V> t;
					t.pack(o);
					t.store(dx + row * dxs + k * V);
				}
			}
		}
	}
	if (!part) return;
	float* pr = part + (static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.y) * 2 * dimp;
#pragma unroll
	for (int i = 0; i < C; ++i)
	{
		const int k = threadIdx.x + i * TPR;
		if (k < nvec)
		{
#pragma unroll
			for (int e = 0; e < V; ++e)
			{
				pr[k * V + e] = aw[i][e];
				pr[dimp + k * V + e] = ab[i][e];
			}
		}
	}
}

// ---- gradient of many rows on 16-byte boundaries: rows arrive by bulk copies, several ahead of the arithmetic --------------
// What bounds the call is how many bytes are on their way per SM; registers that also hold the sums of dw and db have no room for them.
// A ring of whole rows in shared memory, filled by bulk copies (one instruction per row, completion counted on an mbarrier), has.

__device__ __forceinline__ bool row_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t* err_word, uint32_t limit)
{
	const bool filled = tc::mbar_wait(bar, parity, abort_flag, limit);
	if (!filled) tc::report_timeout(err_word, tc::kErrRowWait);
	return filled;
}

// Gradient: a CTA of 256 threads walks groups of R rows; a thread owns NV 16-byte vectors of columns, so dw and db are sums in its
// registers. One barrier per group: both sums of all its rows go through shared memory at once, and whoever has passed it has also
// finished the group before, whose ring stage thread 0 then refills.
constexpr int kRowThreads = 256;
template <typename T, int NV, int R>
__global__ void __launch_bounds__(kRowThreads) layer_norm_backward_rows_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x,
	int64_t xs, const T* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, int64_t dxs,
	float* __restrict__ part, int64_t rows, int dim, int64_t dimp, int stages, uint32_t* err_word, uint32_t wait_limit)
{
	constexpr int V = 16 / sizeof(T), NW = kRowThreads / 32;
	extern __shared__ __align__(128) unsigned char smem[];  // [stages][R][x | dy][dim]
	__shared__ uint64_t full[4];
	__shared__ float red[2][2 * R][NW];
	__shared__ int abort_flag;
	const int bytes = dim * static_cast<int>(sizeof(T)), nvec = dim / V, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	if (threadIdx.x == 0)
	{
		abort_flag = 0;
		for (int i = 0; i < 4; ++i) tc::mbar_init(tc::smem_u32(&full[i]), 1);
		tc::fence_mbar_init();
	}
	__syncthreads();
	const int64_t groups = (rows + R - 1) / R;
	int64_t requests = wait_limit == tc::kSpinLimit ? groups : groups - 1;  // the self-test: a stage that nothing fills
	auto request = [&](int64_t g, int st) {
		const int live = rows - g * R < R ? static_cast<int>(rows - g * R) : R;
		const uint32_t bar = tc::smem_u32(&full[st]);
		tc::mbar_arrive_expect_tx(bar, 2 * live * bytes);
		for (int r = 0; r < live; ++r)
		{
			const uint32_t dst = tc::smem_u32(smem + static_cast<size_t>((st * R + r) * 2) * bytes);
			tc::bulk_load_1d(dst, x + (g * R + r) * xs, bytes, bar);
			tc::bulk_load_1d(dst + bytes, dy + (g * R + r) * dys, bytes, bar);
		}
	};
	if (threadIdx.x == 0)
		for (int i = 0; i < stages && blockIdx.x + static_cast<int64_t>(i) * gridDim.x < requests; ++i) request(blockIdx.x + static_cast<int64_t>(i) * gridDim.x, i);
	const float inv = 1.f / static_cast<float>(dim);
	f2 aw[NV][V / 2], ab[NV][V / 2];
	Pack<T, V> pw[NV];
#pragma unroll
	for (int i = 0; i < NV; ++i)
	{
		const int k = threadIdx.x + i * kRowThreads;
		float one[V];
#pragma unroll
		for (int e = 0; e < V; ++e) one[e] = 1.f;
		pw[i].pack(one);
		if (w && k < nvec) pw[i].load(w + k * V);
#pragma unroll
		for (int e = 0; e < V / 2; ++e) aw[i][e] = ab[i][e] = 0ull;
	}
	float nmu[R], nr[R];
	auto statistics = [&](int64_t g) {
#pragma unroll
		for (int r = 0; r < R; ++r)
		{
			const int64_t row = g * R + r < rows ? g * R + r : rows - 1;
			nmu[r] = mean[row];
			nr[r] = rstd[row];
		}
	};
	if (blockIdx.x < groups) statistics(blockIdx.x);
	int st = 0, phase = 0;
	uint32_t parity = 0;
	for (int64_t g = blockIdx.x; g < groups; g += gridDim.x, phase ^= 1)
	{
		// With xc = x - mu: dw = sum rs (dy xc), t2 = rs mean(w (dy xc)), dx = rs q + xc cx + c0 (cx = -rs^2 t2, c0 = -rs t1). x rs - mu rs in one
		// multiply-add would be off by half a step of mu rs, which an offset common to the row makes large. In f16 the subtraction also
		// widens x (16384 x 3584: 71 us, as a packed addition of its own 80.4). dx does take x cx + (c0 - mu cx), with the rounding of that
		// constant added to q (74.5 us with the subtraction here too).
		float nmean[R], rs[R];
		f2 s1[R], s2[R];
#pragma unroll
		for (int r = 0; r < R; ++r)
		{
			nmean[r] = -nmu[r];
			rs[r] = nr[r];
			s1[r] = s2[r] = 0ull;
		}
		if (g + gridDim.x < groups) statistics(g + gridDim.x);
		const T* stage = reinterpret_cast<const T*>(smem + static_cast<size_t>(st * R * 2) * bytes);
		if (!row_wait(tc::smem_u32(&full[st]), parity, &abort_flag, err_word, wait_limit)) requests = 0;
#pragma unroll
		for (int r = 0; r < R; ++r)
		{
			if (g * R + r >= rows) continue;
			const T* sx = stage + static_cast<size_t>(r) * 2 * dim;
#pragma unroll
			for (int i = 0; i < NV; ++i)
			{
				const int k = threadIdx.x + i * kRowThreads;
				if (k < nvec)
				{
					Pack<T, V> t;
					f2 f[V / 2], d[V / 2], wv[V / 2];
					t.load(sx + k * V);
					unpack_pairs_plus(t, nmean[r], f);
					t.load(sx + dim + k * V);
					unpack_pairs(t, d);
					unpack_pairs(pw[i], wv);
#pragma unroll
					for (int e = 0; e < V / 2; ++e)
					{
						const f2 p = mul2(d[e], f[e]);
						aw[i][e] = fma2(p, both(rs[r]), aw[i][e]);
						ab[i][e] = add2(ab[i][e], d[e]);
						s1[r] = fma2(d[e], wv[e], s1[r]);
						s2[r] = fma2(p, wv[e], s2[r]);
					}
				}
			}
		}
#pragma unroll
		for (int r = 0; r < R; ++r)
		{
			const float a = warp_sum(sum2(s1[r])), c = warp_sum(sum2(s2[r]));
			if (lane == 0)
			{
				red[phase][2 * r][warp] = a;
				red[phase][2 * r + 1][warp] = c;
			}
		}
		__syncthreads();
		const int64_t ahead = g + static_cast<int64_t>(stages - 1) * gridDim.x;  // of the stage that the group before this one has left
		if (threadIdx.x == 0 && g != blockIdx.x && ahead < requests) request(ahead, st == 0 ? stages - 1 : st - 1);
		if (dx)
#pragma unroll
			for (int r = 0; r < R; ++r)
			{
				if (g * R + r >= rows) continue;
				float t1 = 0.f, t2 = 0.f;
#pragma unroll
				for (int i = 0; i < NW; ++i)
				{
					t1 += red[phase][2 * r][i];
					t2 += red[phase][2 * r + 1][i];
				}
				const float cx1 = -rs[r] * (t2 * rs[r] * inv) * rs[r], c0 = -rs[r] * (t1 * inv);
				const float hi = nmean[r] * cx1, sum = hi + c0, part0 = sum - hi;  // -mu cx + c0 = sum + lo
				const float lo = fmaf(nmean[r], cx1, -hi) + ((hi - (sum - part0)) + (c0 - part0));
				const f2 cx = both(cx1), cs = both(sum), cq = both(rs[r]), cl = both(rs[r] != 0.f ? lo / rs[r] : 0.f);
				const T* sx = stage + static_cast<size_t>(r) * 2 * dim;
#pragma unroll
				for (int i = 0; i < NV; ++i)
				{
					const int k = threadIdx.x + i * kRowThreads;
					if (k < nvec)
					{
						Pack<T, V> t;
						f2 f[V / 2], d[V / 2], wv[V / 2];
						float o[V];
						t.load(sx + k * V);
						unpack_pairs(t, f);
						t.load(sx + dim + k * V);
						unpack_pairs(t, d);
						unpack_pairs(pw[i], wv);
#pragma unroll
						for (int e = 0; e < V / 2; ++e)
						{
							const float2 v = unpack2(fma2(fma2(d[e], wv[e], cl), cq, fma2(f[e], cx, cs)));
							o[2 * e] = v.x;
							o[2 * e + 1] = v.y;
						}
						t.pack(o);
						t.store(dx + (g * R + r) * dxs + k * V);
					}
				}
			}
		if (++st == stages)
		{
			st = 0;
			parity ^= 1;
		}
	}
	if (*reinterpret_cast<volatile int*>(&abort_flag))
	{
		// a wait was given up: nothing more was requested, and copies already in flight get time to land before shared memory is released
		for (int i = 0; i < 2000; ++i) __nanosleep(1000);
	}
	if (!part) return;
	float* pr = part + static_cast<int64_t>(blockIdx.x) * 2 * dimp;
#pragma unroll
	for (int i = 0; i < NV; ++i)
	{
		const int k = threadIdx.x + i * kRowThreads;
		if (k < nvec)
		{
#pragma unroll
			for (int e = 0; e < V / 2; e += 2)
			{
				*reinterpret_cast<ulonglong2*>(pr + k * V + 2 * e) = make_ulonglong2(aw[i][e], aw[i][e + 1]);
				*reinterpret_cast<ulonglong2*>(pr + dimp + k * V + 2 * e) = make_ulonglong2(ab[i][e], ab[i][e + 1]);
			}
		}
	}
}

// Rows that do not fit: dx with one CTA per row that reads the row twice, dw and db with one thread per column.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_dx_wide_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
	const T* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, int64_t dxs, int dim)
{
	__shared__ float red[2][8];
	const int64_t row = blockIdx.x;
	const T* xr = x + row * xs;
	const T* dr = dy + row * dys;
	const float mu = mean[row], r = rstd[row];
	float s1 = 0.f, s2 = 0.f;
	for (int i = threadIdx.x; i < dim; i += 256)
	{
		const float q = ldf(dr + i) * (w ? ldf(w + i) : 1.f);
		s1 += q;
		s2 += q * ((ldf(xr + i) - mu) * r);
	}
	const float inv = 1.f / static_cast<float>(dim);
	s1 = row_sum<256>(s1, red[0]) * inv;
	s2 = row_sum<256>(s2, red[1]) * inv;
	for (int i = threadIdx.x; i < dim; i += 256)
	{
		const float q = ldf(dr + i) * (w ? ldf(w + i) : 1.f);
		stf(dx + row * dxs + i, r * (q - s1 - ((ldf(xr + i) - mu) * r) * s2));
	}
}

template <typename T>
__global__ void __launch_bounds__(256) layer_norm_dw_wide_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
	const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part, int64_t rows, int dim, int64_t dimp)
{
	const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
	if (c >= dim) return;
	float aw = 0.f, ab = 0.f;
	for (int64_t row = blockIdx.y; row < rows; row += gridDim.y)
	{
		const float d = ldf(dy + row * dys + c);
		aw += d * ((ldf(x + row * xs + c) - mean[row]) * rstd[row]);
		ab += d;
	}
	float* pr = part + static_cast<int64_t>(blockIdx.y) * 2 * dimp;
	pr[c] = aw;
	pr[dimp + c] = ab;
}

constexpr int kRingBytes = 104 * 1024;   // of a CTA, two of which share an SM
constexpr int kRingMax = 200 * 1024;     // of a CTA that has the SM for itself

// Ring of stages of `unit` bytes each, 64 KB at most (two rows of 8192 fp32 columns, the longest that take it): stages and CTAs per SM.
struct Ring
{
	int stages, ctas;
};
static Ring ring_of(int64_t unit)
{
	static_assert(kRingMax >= 2 * 65536, "two stages at least");
	if (2 * unit <= kRingBytes) return { static_cast<int>(kRingBytes / unit < 4 ? kRingBytes / unit : 4), 2 };
	return { static_cast<int>(kRingMax / unit < 4 ? kRingMax / unit : 4), 1 };
}

// partial rows of dw / db: the workspace holds the larger of what the two forms of the kernel want (a function of the sizes alone)
struct LnPlan
{
	int threads, rows_per_cta, grid, partials;
	bool wide;
	int64_t dimp;
};
static LnPlan ln_backward_plan(int64_t rows, int64_t dim)
{
	LnPlan p;
	p.dimp = cdiv(dim, 4) * 4;
	p.wide = dim > static_cast<int64_t>(kLnMaxThreads) * kLnElems;
	p.threads = ln_threads(dim);
	p.rows_per_cta = p.threads < 128 ? 128 / p.threads : 1;
	// Up to 296 partial rows (148 where a CTA holds one) as few rows each as there are: adding those up is cheaper than walking (16 x 1001
	// columns 4.2 us against 7.0 with 4 rows each, 592 rows 7.3 against 8.0). More only with 4 rows each (1237 rows: 10.3 us, with 2 10.6,
	// with 1 14.4; 5000 x 257: 15, 22, 22).
	const int64_t groups = cdiv(rows, p.rows_per_cta), few = p.rows_per_cta > 1 ? 2 * kNumSMs / p.rows_per_cta : kNumSMs;
	const int64_t fours = cdiv(groups, 4), fill = groups < few ? groups : few;
	const int64_t want = p.wide ? rows : (fours > fill ? fours : fill);
	const int64_t most = p.wide ? 64 : static_cast<int64_t>(kNumSMs) * (512 / (p.threads * p.rows_per_cta));
	p.grid = static_cast<int>(want < most ? want : most);
	p.partials = p.wide ? p.grid : p.grid * p.rows_per_cta;
	return p;
}
// The ring form of the gradient: groups of R rows, so that a stage holds 8 - 32 KB.
struct LnRowsPlan
{
	int r, grid;
	Ring ring;
};
static LnRowsPlan ln_rows_plan(int64_t rows, int64_t row_bytes)
{
	LnRowsPlan p;
	p.r = row_bytes <= 8192 ? 2 : 1;
	p.ring = ring_of(2 * p.r * row_bytes);
	const int64_t groups = cdiv(rows, p.r), most = static_cast<int64_t>(kNumSMs) * p.ring.ctas;
	p.grid = static_cast<int>(groups < most ? groups : most);
	return p;
}
// Where the ring form is taken (rows on 16-byte boundaries). Rows of 2 KB and more: always (f16, 1024 - 8192 columns, ring against registers:
// 16 rows 4.5 - 6.6 us against 7.2 - 16.8, 1184 rows 8.3 - 22.2 against 10.3 - 27.2, 16384 rows 40 - 140 against 40 - 177). Shorter rows leave most
// of its 256 threads idle: only few of them (512 f16 columns: 148 rows 5.1 against 7.6 us, but 16384 rows 38 against 36; 256: 36 against 25).
static bool ln_rows_fit(int64_t rows, int64_t dim, int64_t row_bytes)
{
	return dim <= 8192 && (row_bytes >= 2048 || (row_bytes >= 512 && rows <= 4 * kNumSMs));
}

template <typename T, int V, int ELEMS, int TPR>
static int launch_ln(const T* x, int64_t xs, const T* w, const T* b, T* y, int64_t ys, float* mean, float* rstd, int64_t rows, int dim,
	float eps, cudaStream_t st)
{
	constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
	const int64_t grid = cdiv(rows, ROWS);
	if (grid > 0x7fffffffLL) return B200_ERR_UNSUPPORTED;
	layer_norm_kernel<T, V, ELEMS, TPR, ROWS><<<static_cast<unsigned>(grid), dim3(TPR, ROWS), 0, st>>>(x, xs, w, b, y, ys, mean, rstd, rows, dim, eps);
	B200_LAUNCH_CHECK();
	return B200_OK;
}

template <typename T, int V>
static int layer_norm_v(const T* x, int64_t xs, const T* w, const T* b, T* y, int64_t ys, float* mean, float* rstd, int64_t rows, int dim,
	float eps, cudaStream_t st)
{
	if constexpr (V == 8)
	{
		if (dim > 2560 && rows >= 8 * kNumSMs)
			return with_ln_threads<true>(ln_threads(dim / 2), [&](auto threads) {
				return launch_ln<T, V, 2 * kLnElems, decltype(threads)::value>(x, xs, w, b, y, ys, mean, rstd, rows, dim, eps, st);
			});
	}
	return with_ln_threads<false>(ln_threads(dim), [&](auto threads) {
		return launch_ln<T, V, kLnElems, decltype(threads)::value>(x, xs, w, b, y, ys, mean, rstd, rows, dim, eps, st);
	});
}

template <typename T>
static int layer_norm(const void* xv, int64_t xs, const void* wv, const void* bv, void* yv, int64_t ys, float* mean, float* rstd,
	int64_t rows, int64_t dim, float eps, cudaStream_t st)
{
	constexpr int E = 16 / sizeof(T);
	const T* x = static_cast<const T*>(xv);
	const T* w = static_cast<const T*>(wv);
	const T* b = static_cast<const T*>(bv);
	T* y = static_cast<T*>(yv);
	const bool vec = aligned16(x) && aligned16(w) && aligned16(b) && aligned16(y) && xs % E == 0 && ys % E == 0 && dim % E == 0;
	if (vec) return layer_norm_v<T, E>(x, xs, w, b, y, ys, mean, rstd, rows, static_cast<int>(dim), eps, st);
	return layer_norm_v<T, 1>(x, xs, w, b, y, ys, mean, rstd, rows, static_cast<int>(dim), eps, st);
}

template <typename T, int V, int TPR>
static int launch_ln_backward(const LnPlan& p, const T* dy, int64_t dys, const T* x, int64_t xs, const T* w, const float* mean,
	const float* rstd, T* dx, int64_t dxs, float* part, int64_t rows, int dim, cudaStream_t st)
{
	constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
	layer_norm_backward_kernel<T, V, TPR, ROWS><<<static_cast<unsigned>(p.grid), dim3(TPR, ROWS), 0, st>>>(dy, dys, x, xs, w, mean, rstd, dx,
		dxs, part, rows, dim, p.dimp);
	B200_LAUNCH_CHECK();
	return B200_OK;
}

template <typename T, int V>
static int layer_norm_backward_v(const LnPlan& p, const T* dy, int64_t dys, const T* x, int64_t xs, const T* w, const float* mean,
	const float* rstd, T* dx, int64_t dxs, float* part, int64_t rows, int dim, cudaStream_t st)
{
	if constexpr (V > 1)  // aligned rows that are not short take the ring: one warp, or two (f16)
	{
		if constexpr (sizeof(T) == 2)
			if (p.threads == 64) return launch_ln_backward<T, V, 64>(p, dy, dys, x, xs, w, mean, rstd, dx, dxs, part, rows, dim, st);
		return launch_ln_backward<T, V, 32>(p, dy, dys, x, xs, w, mean, rstd, dx, dxs, part, rows, dim, st);
	}
	else return with_ln_threads<false>(p.threads, [&](auto threads) {
		return launch_ln_backward<T, V, decltype(threads)::value>(p, dy, dys, x, xs, w, mean, rstd, dx, dxs, part, rows, dim, st);
	});
}

// The poll limit of the ring's waits; another one (b200_debug_layer_norm_backward_starved) also leaves out the last group's copies.
static thread_local uint32_t g_row_wait_limit = tc::kSpinLimit;

template <typename T, int NV, int R>
static int launch_ln_rows_backward(const LnRowsPlan& p, const T* dy, int64_t dys, const T* x, int64_t xs, const T* w, const float* mean,
	const float* rstd, T* dx, int64_t dxs, float* part, int64_t rows, int dim, int64_t dimp, cudaStream_t st)
{
	static bool done[64];
	B200_CUDA_TRY(allow_dynamic_smem(layer_norm_backward_rows_kernel<T, NV, R>, kRingMax, done));
	const size_t bytes = static_cast<size_t>(p.ring.stages) * 2 * R * dim * sizeof(T);
	layer_norm_backward_rows_kernel<T, NV, R><<<p.grid, kRowThreads, bytes, st>>>(dy, dys, x, xs, w, mean, rstd, dx, dxs, part, rows, dim, dimp,
		p.ring.stages, device_error_word(), g_row_wait_limit);
	B200_LAUNCH_CHECK();
	return B200_OK;
}

template <typename T>
static int layer_norm_backward(const void* dyv, int64_t dys, const void* xv, int64_t xs, const void* wv, const float* mean, const float* rstd,
	void* dxv, int64_t dxs, float* dw, float* db, int64_t rows, int64_t dim, float* part, cudaStream_t st)
{
	constexpr int E = 16 / sizeof(T);
	const T* dy = static_cast<const T*>(dyv);
	const T* x = static_cast<const T*>(xv);
	const T* w = static_cast<const T*>(wv);
	T* dx = static_cast<T*>(dxv);
	const LnPlan p = ln_backward_plan(rows, dim);
	const int d = static_cast<int>(dim);
	int rc = B200_OK, partials = p.partials;
	if (p.wide)
	{
		if (rows > 0x7fffffffLL) return B200_ERR_UNSUPPORTED;
		if (dx)
		{
			layer_norm_dx_wide_kernel<T><<<static_cast<unsigned>(rows), 256, 0, st>>>(dy, dys, x, xs, w, mean, rstd, dx, dxs, d);
			B200_LAUNCH_CHECK();
		}
		if (part)
		{
			layer_norm_dw_wide_kernel<T><<<dim3(static_cast<unsigned>(cdiv(dim, 256)), static_cast<unsigned>(p.grid)), 256, 0, st>>>(dy, dys, x,
				xs, mean, rstd, part, rows, d, p.dimp);
			B200_LAUNCH_CHECK();
		}
	}
	else
	{
		const bool vec = aligned16(dy) && aligned16(x) && aligned16(w) && aligned16(dx) && dys % E == 0 && xs % E == 0 &&
			(!dx || dxs % E == 0) && dim % E == 0;
		const int64_t row_bytes = dim * static_cast<int64_t>(sizeof(T));
		if (vec && ln_rows_fit(rows, dim, row_bytes))
		{
			const LnRowsPlan rp = ln_rows_plan(rows, row_bytes);
			const int nv = static_cast<int>(cdiv(dim, static_cast<int64_t>(kRowThreads) * E));
#define B200_LN_ROWS(NV, R) launch_ln_rows_backward<T, NV, R>(rp, dy, dys, x, xs, w, mean, rstd, dx, dxs, part, rows, d, p.dimp, st)
			if (rp.r == 2) rc = nv == 1 ? B200_LN_ROWS(1, 2) : B200_LN_ROWS(2, 2);
			else if (nv <= 3) rc = B200_LN_ROWS(3, 1);
			else if (sizeof(T) == 2 || nv == 4) rc = B200_LN_ROWS(4, 1);
			else if constexpr (sizeof(T) == 4) rc = B200_LN_ROWS(8, 1);
#undef B200_LN_ROWS
			partials = rp.grid;
		}
		else rc = vec ? layer_norm_backward_v<T, E>(p, dy, dys, x, xs, w, mean, rstd, dx, dxs, part, rows, d, st)
			: layer_norm_backward_v<T, 1>(p, dy, dys, x, xs, w, mean, rstd, dx, dxs, part, rows, d, st);
	}
	if (rc != B200_OK || !part) return rc;
	ReduceJobs jobs = {};
	int n = 0;
	if (dw) jobs.j[n++] = { part, 2 * p.dimp, dim, dw, 1 };
	if (db) jobs.j[n++] = { part + p.dimp, 2 * p.dimp, dim, db, 1 };
	return column_reduce(jobs, n, partials, st);
}

}  // namespace b200

using namespace b200;

extern "C" int b200_layer_norm(int dtype, const void* x, int64_t x_stride, const void* w, const void* b, void* y, int64_t y_stride,
	float* mean, float* rstd, int64_t rows, int64_t dim, float eps, void* stream)
{
	if (!x || !y) return B200_ERR_NULL;
	if (rows < 0 || dim <= 0 || x_stride < dim || y_stride < dim) return B200_ERR_BAD_SHAPE;
	if (dtype != B200_F16 && dtype != B200_F32) return B200_ERR_UNSUPPORTED;
	if (dim > 0x3fffffffLL) return B200_ERR_UNSUPPORTED;
	if (rows == 0) return B200_OK;
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	if (dtype == B200_F16) return layer_norm<__half>(x, x_stride, w, b, y, y_stride, mean, rstd, rows, dim, eps, st);
	return layer_norm<float>(x, x_stride, w, b, y, y_stride, mean, rstd, rows, dim, eps, st);
}

extern "C" size_t b200_layer_norm_backward_workspace_bytes(int64_t rows, int64_t dim)
{
	if (rows <= 0 || dim <= 0 || dim > 0x3fffffffLL) return 0;
	const LnPlan p = ln_backward_plan(rows, dim);
	const int64_t most = ln_rows_fit(rows, dim, 4 * dim) ? 2 * kNumSMs : 0;  // partial rows of the ring form
	return static_cast<size_t>(p.partials < most ? most : p.partials) * 2 * static_cast<size_t>(p.dimp) * sizeof(float);
}

extern "C" int b200_layer_norm_backward(int dtype, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* w,
	const float* mean, const float* rstd, void* dx, int64_t dx_stride, float* dw, float* db, int64_t rows, int64_t dim, void* workspace,
	size_t workspace_bytes, void* stream)
{
	if (!dy || !x || !mean || !rstd || (!dx && !dw && !db)) return B200_ERR_NULL;
	if (rows < 0 || dim <= 0 || dy_stride < dim || x_stride < dim || (dx && dx_stride < dim)) return B200_ERR_BAD_SHAPE;
	if (dtype != B200_F16 && dtype != B200_F32) return B200_ERR_UNSUPPORTED;
	if (dim > 0x3fffffffLL) return B200_ERR_UNSUPPORTED;
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	if (rows == 0)
	{
		// the sum over no rows
		if (dw) B200_CUDA_TRY(cudaMemsetAsync(dw, 0, static_cast<size_t>(dim) * sizeof(float), st));
		if (db) B200_CUDA_TRY(cudaMemsetAsync(db, 0, static_cast<size_t>(dim) * sizeof(float), st));
		return B200_OK;
	}
	float* part = nullptr;
	if (dw || db)
	{
		if (!workspace || workspace_bytes < b200_layer_norm_backward_workspace_bytes(rows, dim)) return B200_ERR_WORKSPACE;
		if (!aligned16(workspace)) return B200_ERR_MISALIGNED;
		part = static_cast<float*>(workspace);
	}
	if (dtype == B200_F16)
		return layer_norm_backward<__half>(dy, dy_stride, x, x_stride, w, mean, rstd, dx, dx_stride, dw, db, rows, dim, part, st);
	return layer_norm_backward<float>(dy, dy_stride, x, x_stride, w, mean, rstd, dx, dx_stride, dw, db, rows, dim, part, st);
}

extern "C" int b200_debug_layer_norm_backward_starved(const void* dy, const void* x, const float* mean, const float* rstd, void* dx, int64_t rows,
	int64_t dim, uint32_t spin_limit, void* stream)
{
	if (!dy || !x || !mean || !rstd || !dx) return B200_ERR_NULL;
	if (rows <= 0 || dim < 1024 || dim > 8192 || dim % 8 != 0 || spin_limit == 0 || spin_limit >= tc::kSpinLimit) return B200_ERR_BAD_SHAPE;
	if (!aligned16(dy) || !aligned16(x) || !aligned16(dx)) return B200_ERR_MISALIGNED;
	g_row_wait_limit = spin_limit;
	const int rc = layer_norm_backward<__half>(dy, dim, x, dim, nullptr, mean, rstd, dx, dim, nullptr, nullptr, rows, dim, nullptr,
		static_cast<cudaStream_t>(stream));
	g_row_wait_limit = tc::kSpinLimit;
	return rc;
}
