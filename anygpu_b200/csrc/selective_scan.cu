// Selective scan with a decay per channel and state, whole sequences and single tokens:
//   h_t[n] = exp(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n],  y_t = (sum_n C_t[n] h_t[n] + D x_t) silu(z_t)   per channel
// The decay differs in every (channel, state), so nothing here is a matrix product: per (token, channel, state) it takes one
// exponential and four multiply-adds, and the exponentials (16 per clock and SM) bound it, not the bytes.
//
// LPC lanes share a channel and own 4 states each, in registers as two packed pairs. A CTA walks its channels in tiles of TT tokens with
// two kinds of warps, because the two kinds of work wait for different things and hide each other's latency when they run side by
// side (8192 x 4096 x 16: 267 us with the same warps doing both in turn, 228 us so; 230 with step sizes to two half steps):
//   * loading warps bring the activations (neighbouring threads, neighbouring channels of a token: a warp that loaded the 16 bytes of its
//     own channels token by token touched 32 cache lines per access, and the memory pipe was half busy with that), and leave
//     (delta, delta x) per (channel, token) and the rows of B and C in shared memory, one tile ahead; one tile behind they apply skip
//     and gate to the sums and store the outputs;
//   * state warps own 32 / LPC channels each and run the recurrence; the sum over n leaves the lanes by a butterfly over four tokens at
//     once. What bounds them beside the exponentials is the traffic between shared memory and registers, so the lanes are numbered for
//     it (Lanes).
// Both meet at one barrier per tile; the shared buffers are double.
#include <type_traits>

#include "selective_scan.cuh"

namespace b200 {

using namespace sscan;

template <typename T, int LPC>
struct ForwardTile
{
	static constexpr int CW = warp_channels(LPC);
	static constexpr int EPT = CW < 8 ? CW : 8;   // channels of one token in a piece that a loading thread handles
	static constexpr int LPT = CW / EPT;          // pieces per token and state warp
	static constexpr int TT = 32 / LPT;           // tokens: 32 pieces per state warp
	static constexpr int NP = LPC * kStates;      // padded states
	// rows of a channel are padded so that what is read or written together lies in different banks
	static constexpr int PS = TT + 1, YS = TT + 4;
	static constexpr int up16(int v) { return (v + 15) / 16 * 16; }
	static constexpr int P = CW * PS * 8;         // (delta, u)
	// a state warp's part of a buffer; 24 bytes past a multiple of 128, which keeps apart what neighbouring threads write to
	static constexpr int WARP = (P + CW * YS * 4 + 103) / 128 * 128 + 24;
	static constexpr int BC = 2 * TT * NP * 4;    // B | C
	static constexpr int buffer(int warps) { return up16(warps * WARP) + BC; }
	// 32 pieces of one activation; x and dt of two tiles on their way to the steps, x and z of two on their way to the outputs
	static constexpr int RAW1 = 32 * (EPT * static_cast<int>(sizeof(T)) < 4 ? 4 : EPT * static_cast<int>(sizeof(T)));
	static constexpr int bytes(int warps) { return 2 * buffer(warps) + up16(2 * warps * CW * 4) + 8 * warps * RAW1; }
};
constexpr int kForwardWarps = 7;                           // state warps of a CTA at most: two CTAs of 14 warps leave 72 registers per thread
constexpr int kForwardThreads = 2 * 32 * kForwardWarps;  // as many loading warps as state warps

// MODE 0: outputs. MODE 1: only what a token segment does to the state, for the segments before the last: the state it ends in from
// zero (slot seg + 1 of seg_state) and the sum of its steps (seg_dsum), and slot 0 = the initial state. The kernel of mode 0
// then enters segment s with  h <- exp(A dsum_q) h + seg_state_{q+1}, q = 0 .. s-1, from slot 0.
template <typename T, int LPC, Access VEC, int MODE>
__global__ void __launch_bounds__(kForwardThreads, 2) selective_scan_kernel(const Inputs in, T* __restrict__ y, int64_t ys, float* fin,
	float* __restrict__ ckpt, float* __restrict__ seg_state, float* __restrict__ seg_dsum, int seg_tokens, int nseg, int warps /* state warps */)
{
	using F = ForwardTile<T, LPC>;
	constexpr int CW = F::CW, EPT = F::EPT, LPT = F::LPT, TT = F::TT, NP = F::NP, PS = F::PS, YS = F::YS;
	constexpr bool EXACT = sizeof(T) == 4;  // decay_2
	extern __shared__ __align__(16) unsigned char smem[];
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	const int buffer = F::buffer(warps), bc_at = F::up16(warps * F::WARP);
	float* s_par = reinterpret_cast<float*>(smem + 2 * buffer);  // [dt_bias | D][warps * CW]
	const int g = blockIdx.x / in.nbg;
	const int c0 = g * in.dpg + (blockIdx.x - g * in.nbg) * warps * CW;  // the CTA's first channel
	const int cend = (g + 1) * in.dpg;
	const int64_t b = blockIdx.y;
	const int seg = blockIdx.z;
	const int64_t t_begin = static_cast<int64_t>(seg) * seg_tokens;
	const int64_t t_end = t_begin + seg_tokens < in.seqlen ? t_begin + seg_tokens : in.seqlen;
	const int N = in.N;
	for (int i = threadIdx.x; i < warps * CW; i += blockDim.x)
	{
		const bool ok = c0 + i < cend;
		s_par[i] = in.bias && ok ? in.bias[c0 + i] : 0.f;
		s_par[warps * CW + i] = MODE == 0 && in.D && ok ? in.D[c0 + i] : 0.f;
	}
	__syncthreads();

	if (warp >= warps)
	{
		// ================================= loading warps =================================================================
		// A thread handles one piece of every tile: channels [lc, lc + EPT) of token lt. The activations travel by asynchronous copies
		// through slots that only this thread reads: [steps: x, dt | outputs: x, z][2 buffers].
		const int id = threadIdx.x - warps * 32, lt = id / (warps * LPT), lc = id % (warps * LPT) * EPT, cn = cend - (c0 + lc);
		const T* xp = static_cast<const T*>(in.x) + b * in.seqlen * in.xs + c0 + lc;
		const T* dp = static_cast<const T*>(in.dt) + b * in.seqlen * in.dts + c0 + lc;
		const T* zp = in.z ? static_cast<const T*>(in.z) + b * in.seqlen * in.zs + c0 + lc : nullptr;
		T* yp = y + b * in.seqlen * ys + c0 + lc;
		const T* Bp = static_cast<const T*>(in.B) + b * in.seqlen * in.Bs + static_cast<int64_t>(g) * N;
		const T* Cp = static_cast<const T*>(in.C) + b * in.seqlen * in.Cs + static_cast<int64_t>(g) * N;
		unsigned char* raw = smem + 2 * buffer + F::up16(2 * warps * CW * 4) + id / 32 * F::RAW1;
		auto slot = [&](int what, int buf) { return raw + (what * 2 + buf) * warps * F::RAW1; };
		unsigned char* mine_s = smem + lc / CW * F::WARP;
		float2* t_p = reinterpret_cast<float2*>(mine_s) + lc % CW * PS + lt;
		const float* t_y = reinterpret_cast<const float*>(mine_s + F::P) + lc % CW * YS + lt;
		const float* t_bias = s_par + lc;
		const float* t_skip = s_par + warps * CW + lc;
		RowsBC<T, NP, TT, MODE == 0 ? 2 : 1> bc(id, warps * 32);
		const bool vec_bc = in.vec_bc;
		// a missing token or channel: an address inside the tensor, from which nothing is read
		auto load = [&](int what, int buf, const T* p, int64_t stride, int64_t t) {
			const bool ok = t < t_end && cn > 0;
			raw_load<T, EPT, VEC>(slot(what, buf), ok ? p + t * stride : p - lc, ok ? cn : 0, lane);
		};
		auto fetch = [&](int64_t t0, int buf) {  // for the steps
			load(0, buf, xp, in.xs, t0 + lt);
			load(1, buf, dp, in.dts, t0 + lt);
			bc.fetch(vec_bc, in, Bp, Cp, t0, t_end);
		};
		auto fetch_outputs = [&](int64_t t0, int buf) {
			load(2, buf, xp, in.xs, t0 + lt);
			if (zp) load(3, buf, zp, in.zs, t0 + lt);
		};
		auto prepare = [&](int64_t t0, int buf) {
			float xv[EPT], dv[EPT];
			raw_read<T, EPT>(slot(0, buf), xv, lane);
			raw_read<T, EPT>(slot(1, buf), dv, lane);
#pragma unroll
			for (int e = 0; e < EPT; ++e) dv[e] += t_bias[e];
			if (in.softplus) softplus_n<EPT>(dv);
			const int have = t0 + lt < t_end ? cn : 0;
			float2* p = reinterpret_cast<float2*>(reinterpret_cast<unsigned char*>(t_p) + buf * buffer);
#pragma unroll
			for (int e = 0; e < EPT; ++e)
			{
				const float dl = e < have ? dv[e] : 0.f;  // a step of zero leaves the state as it is
				p[e * PS] = make_float2(dl, dl * xv[e]);
			}
			bc.store(vec_bc, in, Bp, Cp, t0, t_end, reinterpret_cast<float*>(smem + buf * buffer + bc_at));
		};
		auto finish = [&](int64_t t0, int buf) {
			if (t0 + lt >= t_end || cn <= 0) return;
			const float* sy = reinterpret_cast<const float*>(reinterpret_cast<const unsigned char*>(t_y) + buf * buffer);
			float o[EPT], xv[EPT];
			raw_read<T, EPT>(slot(2, buf), xv, lane);
#pragma unroll
			for (int e = 0; e < EPT; ++e) o[e] = sy[e * YS] + t_skip[e] * xv[e];
			if (zp)
			{
				float zv[EPT], sg[EPT];
				raw_read<T, EPT>(slot(3, buf), zv, lane);
				sigmoid_n<EPT, EXACT>(zv, sg);
#pragma unroll
				for (int e = 0; e < EPT; ++e) o[e] *= zv[e] * sg[e];
			}
			store_frag<T, EPT, VEC>(o, yp + (t0 + lt) * ys, cn);
		};
		auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
		fetch(t_begin, 0);
		commit();
		asm volatile("cp.async.wait_group 0;" ::: "memory");
		prepare(t_begin, 0);
		fetch(t_begin + TT, 1);
		if (MODE == 0) fetch_outputs(t_begin, 0);
		commit();
		__syncthreads();
		int buf = 0;
		for (int64_t t0 = t_begin; t0 < t_end; t0 += TT, buf ^= 1)
		{
			// while the state warps are at tile t0
			asm volatile("cp.async.wait_group 0;" ::: "memory");
			if (t0 + TT < t_end) prepare(t0 + TT, buf ^ 1);
			if (t0 + 2 * TT < t_end) fetch(t0 + 2 * TT, buf);
			if (MODE == 0 && t0 > t_begin) finish(t0 - TT, buf ^ 1);
			if (MODE == 0 && t0 + TT < t_end) fetch_outputs(t0 + TT, buf ^ 1);
			commit();
			__syncthreads();
		}
		asm volatile("cp.async.wait_group 0;" ::: "memory");
		if (MODE == 0) finish(t_begin + (t_end - 1 - t_begin) / TT * TT, buf ^ 1);
		return;
	}

	// ===================================== state warps =====================================================================
	const int sub = Lanes<LPC>::sub(lane), cl = Lanes<LPC>::cl(lane), n0 = sub * kStates, c = c0 + warp * CW + cl;
	const bool mine = c < cend, vec4 = N % 4 == 0;
	const int64_t row = (b * in.dim + c) * N;
	const int64_t slots = static_cast<int64_t>(gridDim.y) * in.dim * N;  // one slot of seg_state
	f2 a2[2] = { 0ull, 0ull }, h[2] = { 0ull, 0ull };
	float dsum = 0.f;
	if (mine)
	{
		float av[kStates];
		load_decay(av, in.A + static_cast<int64_t>(c) * N, in.a_is_log, n0, N);
		a2[0] = pack2(av[0], av[1]);
		a2[1] = pack2(av[2], av[3]);
		if (MODE == 1)
		{
			if (seg == 0)
			{
				float i0[kStates] = { 0.f, 0.f, 0.f, 0.f };
				if (in.init) load_states(vec4, i0, in.init + row, n0, N);
				store_states(vec4, i0, seg_state + row, n0, N);
			}
		}
		else if (nseg > 1)
		{
			load_states2(vec4, h, seg_state + row, n0, N);
#pragma unroll 8  // the loads of eight segments at a time
			for (int q = 0; q < seg; ++q)
			{
				f2 add[2];
				load_states2(vec4, add, seg_state + (q + 1) * slots + row, n0, N);
				const f2 ds = both(seg_dsum[(static_cast<int64_t>(q) * gridDim.y + b) * in.dim + c]);
#pragma unroll
				for (int i = 0; i < 2; ++i) h[i] = fma2(decay_2<true>(mul2(ds, a2[i])), h[i], add[i]);
			}
		}
		else if (in.init) load_states2(vec4, h, in.init + row, n0, N);
	}
	__syncthreads();
	int buf = 0;
	for (int64_t t0 = t_begin; t0 < t_end; t0 += TT, buf ^= 1)
	{
		const float2* s_p = reinterpret_cast<const float2*>(smem + buf * buffer + warp * F::WARP) + cl * PS;
		float* s_y = reinterpret_cast<float*>(smem + buf * buffer + warp * F::WARP + F::P) + cl * YS + TokenSum<LPC>::first(sub);
		const float* s_B = reinterpret_cast<const float*>(smem + buf * buffer + bc_at) + n0;
		const float* s_C = s_B + TT * NP;
		// Unrolled, and the results stay in registers until the tile is through: a store to shared memory would hold back the loads of the
		// next tokens, and with them the arithmetic that hides the latency of the exponentials and the shuffles.
		float tot[TT / 4][TokenSum<LPC>::COUNT];
		constexpr int kGroups = MODE == 0 ? TT / 4 : 2;
#pragma unroll kGroups
		for (int t4 = 0; t4 < TT; t4 += 4)
		{
			if (MODE == 0 && t4 % kTok == 0)
				if (ckpt && mine && (TT >= kTok || t0 % kTok == 0) && t0 + t4 < t_end)
					store_states2(vec4, h, ckpt + ((b * cdiv(in.seqlen, kTok) + (t0 + t4) / kTok) * in.dim + c) * N, n0, N);
			float acc[4];
#pragma unroll
			for (int j = 0; j < 4; ++j)
			{
				const float2 p = s_p[t4 + j];
				const f2 dl = both(p.x), u = both(p.y);
				const ulonglong2 Bv = *reinterpret_cast<const ulonglong2*>(s_B + (t4 + j) * NP);
				h[0] = fma2(decay_2<EXACT>(mul2(dl, a2[0])), h[0], mul2(u, Bv.x));
				h[1] = fma2(decay_2<EXACT>(mul2(dl, a2[1])), h[1], mul2(u, Bv.y));
				if (MODE == 0)
				{
					const ulonglong2 Cv = *reinterpret_cast<const ulonglong2*>(s_C + (t4 + j) * NP);
					acc[j] = sum2(fma2(h[1], Cv.y, mul2(h[0], Cv.x)));
				}
				else dsum += p.x;
			}
			if (MODE == 0) TokenSum<LPC>::run(acc, sub, tot[t4 / 4]);
		}
		if (MODE == 0 && TokenSum<LPC>::owner(sub))
#pragma unroll
			for (int i = 0; i < TT / 4; ++i)
#pragma unroll
				for (int j = 0; j < TokenSum<LPC>::COUNT; ++j) s_y[i * 4 + j] = tot[i][j];
		__syncthreads();
	}
	if (!mine) return;
	if (MODE == 1)
	{
		store_states2(vec4, h, seg_state + (seg + 1) * slots + row, n0, N);
		if (sub == 0) seg_dsum[(static_cast<int64_t>(seg) * gridDim.y + b) * in.dim + c] = dsum;
	}
	else if (fin && seg == nseg - 1) store_states2(vec4, h, fin + row, n0, N);
}

// One token. A thread owns 4 states of one channel for RB batch entries, whose states it requests before it uses the first: the kernel
// streams 8 bytes of state per (channel, state) and everything else is small next to that. VEC: 16-byte states and 4-element rows of B
// and C (d_state, strides and bases multiples of 4 elements).
template <typename T, int RB, bool VEC>
__global__ void __launch_bounds__(128) selective_scan_update_kernel(float* __restrict__ state, const Inputs in, T* __restrict__ y, int64_t ys,
	int64_t batch, int lpc)
{
	const int sub = threadIdx.x % lpc;
	const int64_t c = static_cast<int64_t>(blockIdx.x) * (128 / lpc) + threadIdx.x / lpc;
	const int64_t b0 = static_cast<int64_t>(blockIdx.y) * RB;
	const bool mine = c < in.dim;
	const int64_t cc = mine ? c : in.dim - 1;  // surplus lanes walk along (the shuffles need them) and write nothing
	const int N = in.N, n0 = sub * kStates;
	const int g = static_cast<int>(cc / in.dpg);
	float h[RB][kStates], xv[RB], dv[RB], zv[RB];
	Pack<T, 4> pB[RB], pC[RB];
	auto entry = [&](int r) { return b0 + r < batch ? b0 + r : batch - 1; };
#pragma unroll
	for (int r = 0; r < RB; ++r) load_states(VEC, h[r], state + (entry(r) * in.dim + cc) * N, n0, N);
#pragma unroll
	for (int r = 0; r < RB; ++r)
	{
		const int64_t b = entry(r);
		xv[r] = ldf(static_cast<const T*>(in.x) + b * in.xs + cc);
		dv[r] = ldf(static_cast<const T*>(in.dt) + b * in.dts + cc);
		zv[r] = in.z ? ldf(static_cast<const T*>(in.z) + b * in.zs + cc) : 0.f;
		const T* Br = static_cast<const T*>(in.B) + b * in.Bs + static_cast<int64_t>(g) * N + n0;
		const T* Cr = static_cast<const T*>(in.C) + b * in.Cs + static_cast<int64_t>(g) * N + n0;
		if constexpr (VEC)
		{
			pB[r].bits = pC[r].bits = {};
			if (n0 < N)
			{
				pB[r].load(Br);
				pC[r].load(Cr);
			}
		}
		else
		{
			float f[kStates], q[kStates];
#pragma unroll
			for (int i = 0; i < kStates; ++i)
			{
				f[i] = n0 + i < N ? ldf(Br + i) : 0.f;
				q[i] = n0 + i < N ? ldf(Cr + i) : 0.f;
			}
			pB[r].pack(f);
			pC[r].pack(q);
		}
	}
	float a2[kStates];
	load_states(VEC, a2, in.A + cc * N, n0, N);
#pragma unroll
	for (int i = 0; i < kStates; ++i) a2[i] = n0 + i < N ? decay_unit(a2[i], in.a_is_log) : 0.f;
	const float bias = in.bias ? in.bias[cc] : 0.f, skip = in.D ? in.D[cc] : 0.f;
	float sg[RB];
#pragma unroll
	for (int r = 0; r < RB; ++r) dv[r] += bias;
	if (in.softplus) softplus_n<RB>(dv);
	sigmoid_n<RB, sizeof(T) == 4>(zv, sg);
#pragma unroll
	for (int r = 0; r < RB; ++r)
	{
		const float u = dv[r] * xv[r];
		float acc = 0.f, Bv[kStates], Cv[kStates];
		pB[r].unpack(Bv);
		pC[r].unpack(Cv);
#pragma unroll
		for (int i = 0; i < kStates; i += 2)
		{
			const float2 a = unpack2(decay_2<true>(pack2(dv[r] * a2[i], dv[r] * a2[i + 1])));
			h[r][i] = a.x * h[r][i] + u * Bv[i];
			h[r][i + 1] = a.y * h[r][i + 1] + u * Bv[i + 1];
			acc += h[r][i] * Cv[i] + h[r][i + 1] * Cv[i + 1];
		}
		for (int o = 1; o < lpc; o <<= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
		if (mine && b0 + r < batch)
		{
			store_states(VEC, h[r], state + ((b0 + r) * in.dim + c) * N, n0, N);
			if (sub == 0)
			{
				float o = acc + skip * xv[r];
				if (in.z) o *= zv[r] * sg[r];
				stf(y + (b0 + r) * ys + c, o);
			}
		}
	}
}

// ---- host ------------------------------------------------------------------------------------------------------------

int selective_scan_check(int dtype, const b200_selective_scan_inputs* in)
{
	if (!in || !in->x || !in->dt || !in->A || !in->B || !in->C) return B200_ERR_NULL;
	if (in->batch < 0 || in->seqlen < 0 || in->dim <= 0 || in->ngroups <= 0 || in->d_state <= 0 || in->dim % in->ngroups != 0)
		return B200_ERR_BAD_SHAPE;
	const int64_t gn = in->ngroups * in->d_state;
	if (in->x_stride < in->dim || in->dt_stride < in->dim || in->B_stride < gn || in->C_stride < gn || (in->z && in->z_stride < in->dim))
		return B200_ERR_BAD_SHAPE;
	if (dtype != B200_F16 && dtype != B200_F32) return B200_ERR_UNSUPPORTED;
	if (in->d_state > kMaxState || in->dim > 0x3fffffffLL || in->seqlen > 0x3fffffffLL || in->batch > 65535 || in->ngroups > 65535)
		return B200_ERR_UNSUPPORTED;
	return B200_OK;
}

Inputs selective_scan_params(const b200_selective_scan_inputs* in, int nbg)
{
	Inputs p;
	p.x = in->x; p.dt = in->dt; p.B = in->B; p.C = in->C; p.z = in->z;
	p.xs = in->x_stride; p.dts = in->dt_stride; p.Bs = in->B_stride; p.Cs = in->C_stride; p.zs = in->z_stride;
	p.A = in->A; p.D = in->D; p.bias = in->dt_bias; p.init = in->initial_state;
	p.a_is_log = in->a_is_log; p.softplus = in->dt_softplus;
	p.seqlen = in->seqlen;
	p.dim = static_cast<int>(in->dim);
	p.N = static_cast<int>(in->d_state);
	p.dpg = static_cast<int>(in->dim / in->ngroups);
	p.nbg = nbg;
	p.vec_bc = 0;
	return p;
}

namespace sscan {
static int forward_smem_bytes(int lpc, int warps)
{
	switch (lpc)
	{
	case 1: return ForwardTile<__half, 1>::bytes(warps);
	case 2: return ForwardTile<__half, 2>::bytes(warps);
	case 4: return ForwardTile<__half, 4>::bytes(warps);
	case 8: return ForwardTile<__half, 8>::bytes(warps);
	case 16: return ForwardTile<__half, 16>::bytes(warps);
	default: return ForwardTile<__half, 32>::bytes(warps);
	}
}

// Token segments (multiples of 32 tokens) and state warps per CTA that a small model of the kernels expects to be fastest. Its terms were
// measured in f16 at 16 states: a token takes a warp (base + state warps on its SM) x 6.0 ns forward (base 4.7; 14 and 36 at up to 8 and 4
// states, where a warp holds 16 and 32 channels and a tile is shorter: 4 x 1024 x 2048 x 8 99 -> 74 us) and x 14.6 ns backward (base 14);
// an SM holds 16 warps (fewer where shared memory runs out), a CTA is not divided between SMs, and what its warps share (rows of B and C;
// backward also the joining of dB and dC) counts as 0.1 (forward) or 0.5 (backward) of a warp's work; S segments cost another pass over
// (S - 1) / S of the tokens that takes 0.95 (forward) or 0.3 (backward) of the time per token, and a launch and a prefix over the segments,
// here in units of those 6.0 and 14.6 ns. Examples, one segment against the choice: 1 x 16384 tokens x 520 channels forward 743 -> 119 us;
// 1 x 2048 x 4096 forward and backward 650 -> 416 us; 4 x 2048 x 4096 stays whole.
Split split_work(int64_t batch, int64_t seqlen, int64_t dim, int64_t ngroups, int64_t d_state, bool backward)
{
	const int lpc = lanes_per_channel(d_state);
	const int64_t nw = cdiv(dim / ngroups, warp_channels(lpc));  // warps across a group
	const int64_t rows = batch * ngroups, warps = rows * nw;
	const double base = backward ? 14 : (lpc == 1 ? 36 : (lpc == 2 ? 14 : 4.7)), again = backward ? 0.3 : 0.95,
		launch = backward ? 350 : 880, prefix = backward ? 8 : 20, shared = backward ? 0.5 : 0.1;
	int64_t most = kNumSMs * 16 / warps;
	if (most > cdiv(seqlen, 32)) most = cdiv(seqlen, 32);
	if (most > 128) most = 128;
	Split s = { 1, 1, 1, 1 };
	double best = 0;
	for (int f = 3; f <= 8; ++f)
	{
		const int64_t want = f == 3 ? 1 : most * f / 8;
		if (f > 3 && want < 2) continue;
		const int64_t tok = cdiv(cdiv(seqlen, want), 32) * 32, seg = cdiv(seqlen, tok);
		if (f > 3 && seg < 2) continue;
		for (int w = max_warps(lpc); w >= 1; --w)
		{
			// where one warp holds a group's channels, more of them still share the loading (1 x 2048 x 8 backward: 72 us, with one 77)
			if ((w > nw || w == 1) && nw > 1) continue;
			// 3, 5 and 6 warps load the four quarters of an SM unevenly (1 x 16384 x 520 forward: 136 - 157 us against 117 - 132)
			if (w == 3 || w == 5 || w == 6 || (!backward && w > kForwardWarps)) continue;
			const int64_t ctas = rows * cdiv(nw, w) * seg, fit = 232448 / ((backward ? backward_smem_bytes(lpc, w) : forward_smem_bytes(lpc, w)) + 1024);
			const int64_t per_sm = fit < 16 / w ? (fit > 0 ? fit : 1) : 16 / w;
			const int64_t waves = cdiv(ctas, kNumSMs * per_sm), busy = cdiv(ctas, kNumSMs);
			const double load = (base + static_cast<double>((busy < per_sm ? busy : per_sm) * w)) * (1 + shared / w);
			double cost = static_cast<double>(waves * tok) * load;
			if (seg > 1) cost += cost * again * static_cast<double>(seg - 1) / static_cast<double>(seg) + launch + prefix * static_cast<double>(seg);
			if (best == 0 || cost < best)
			{
				best = cost;
				s = { w, static_cast<int>(cdiv(nw, w)), static_cast<int>(seg), static_cast<int>(tok) };
			}
		}
	}
	return s;
}
}  // namespace sscan

template <typename T, int LPC, Access VEC, int MODE>
static int launch_scan_kernel(const Split& sp, const dim3& g, const Inputs& p, T* y, int64_t ys, float* fin, float* ckpt, float* seg_state,
	float* seg_dsum, cudaStream_t st)
{
	static bool done[64];
	B200_CUDA_TRY(allow_dynamic_smem(selective_scan_kernel<T, LPC, VEC, MODE>, ForwardTile<T, LPC>::bytes(kForwardWarps), done));
	selective_scan_kernel<T, LPC, VEC, MODE><<<g, 2 * 32 * sp.warps, ForwardTile<T, LPC>::bytes(sp.warps), st>>>(p, y, ys, fin,
		ckpt, seg_state, seg_dsum, sp.seg_tokens, sp.nseg, sp.warps);
	B200_LAUNCH_CHECK();
	return B200_OK;
}

template <typename T, int LPC>
static int launch_scan(const b200_selective_scan_inputs* in, const Split& sp, T* y, int64_t ys, float* fin, float* ckpt, float* ws, cudaStream_t st)
{
	constexpr int EPT = ForwardTile<T, LPC>::EPT;
	Inputs p = selective_scan_params(in, sp.nbg);
	p.vec_bc = RowsBC<T, ForwardTile<T, LPC>::NP, ForwardTile<T, LPC>::TT, 2>::aligned(in);
	const bool vec = p.dpg % EPT == 0 && frag_aligned<T, EPT>(p.x, p.xs) && frag_aligned<T, EPT>(p.dt, p.dts) && frag_aligned<T, EPT>(p.z, p.zs) &&
		frag_aligned<T, EPT>(y, ys);
	const bool words = sizeof(T) == 2 && p.dpg % 2 == 0 && word_aligned(p.x, p.xs) && word_aligned(p.dt, p.dts) && word_aligned(p.z, p.zs) &&
		word_aligned(y, ys);
	const dim3 g(static_cast<unsigned>(in->ngroups * p.nbg), static_cast<unsigned>(in->batch), static_cast<unsigned>(sp.nseg));
	float* seg_state = ws;
	float* seg_dsum = ws ? ws + static_cast<int64_t>(sp.nseg) * in->batch * in->dim * in->d_state : nullptr;
	auto run = [&](auto access) {
		constexpr Access VEC = decltype(access)::value;
		if (sp.nseg > 1)
		{
			const dim3 g1(g.x, g.y, g.z - 1);
			const int rc = launch_scan_kernel<T, LPC, VEC, 1>(sp, g1, p, y, ys, fin, ckpt, seg_state, seg_dsum, st);
			if (rc != B200_OK) return rc;
		}
		return launch_scan_kernel<T, LPC, VEC, 0>(sp, g, p, y, ys, fin, ckpt, seg_state, seg_dsum, st);
	};
	if (vec) return run(std::integral_constant<Access, kVectors>{});
	if constexpr (sizeof(T) == 2)
		if (words) return run(std::integral_constant<Access, kWords>{});
	return run(std::integral_constant<Access, kSingle>{});
}

template <typename T>
static int scan(const b200_selective_scan_inputs* in, void* yv, int64_t ys, float* fin, float* ckpt, float* ws, const Split& sp,
	cudaStream_t st)
{
	T* y = static_cast<T*>(yv);
	switch (lanes_per_channel(in->d_state))
	{
	case 1: return launch_scan<T, 1>(in, sp, y, ys, fin, ckpt, ws, st);
	case 2: return launch_scan<T, 2>(in, sp, y, ys, fin, ckpt, ws, st);
	case 4: return launch_scan<T, 4>(in, sp, y, ys, fin, ckpt, ws, st);
	case 8: return launch_scan<T, 8>(in, sp, y, ys, fin, ckpt, ws, st);
	case 16: return launch_scan<T, 16>(in, sp, y, ys, fin, ckpt, ws, st);
	default: return launch_scan<T, 32>(in, sp, y, ys, fin, ckpt, ws, st);
	}
}

template <typename T, int RB>
static void launch_update(float* state, const Inputs& p, T* y, int64_t ys, int64_t batch, int lpc, cudaStream_t st)
{
	const dim3 g(static_cast<unsigned>(cdiv(p.dim, 128 / lpc)), static_cast<unsigned>(cdiv(batch, RB)));
	auto al = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & (4 * sizeof(T) - 1)) == 0; };
	const bool vec = p.N % 4 == 0 && al(p.B) && al(p.C) && p.Bs % 4 == 0 && p.Cs % 4 == 0 && aligned16(p.A);
	if (vec) selective_scan_update_kernel<T, RB, true><<<g, 128, 0, st>>>(state, p, y, ys, batch, lpc);
	else selective_scan_update_kernel<T, RB, false><<<g, 128, 0, st>>>(state, p, y, ys, batch, lpc);
}

template <typename T>
static int scan_update(float* state, const Inputs& p, void* yv, int64_t ys, int64_t batch, cudaStream_t st)
{
	const int lpc = lanes_per_channel(p.N);
	T* y = static_cast<T*>(yv);
	constexpr int RB = 4;
	// several entries per thread share A and keep more loads in flight; not where that would leave SMs without work (16 states, one entry
	// against four per thread: 8 x 4096 3.9 us against 4.2, 16 x 4096 5.9 against 5.0, 128 x 4096 29 against 24)
	if (batch * cdiv(p.dim, 128 / lpc) >= kNumSMs * 10LL) launch_update<T, RB>(state, p, y, ys, batch, lpc, st);
	else launch_update<T, 1>(state, p, y, ys, batch, lpc, st);
	B200_LAUNCH_CHECK();
	return B200_OK;
}

}  // namespace b200

using namespace b200;

extern "C" size_t b200_selective_scan_workspace_bytes(int64_t batch, int64_t seqlen, int64_t dim, int64_t ngroups, int64_t d_state)
{
	if (batch <= 0 || seqlen <= 0 || dim <= 0 || ngroups <= 0 || d_state <= 0 || dim % ngroups != 0 || d_state > kMaxState) return 0;
	const int s = split_work(batch, seqlen, dim, ngroups, d_state, false).nseg;
	if (s == 1) return 0;
	return (static_cast<size_t>(s) * batch * dim * d_state + static_cast<size_t>(s - 1) * batch * dim) * sizeof(float);
}

extern "C" size_t b200_selective_scan_checkpoint_bytes(int64_t batch, int64_t seqlen, int64_t dim, int64_t d_state)
{
	if (batch <= 0 || seqlen <= 0 || dim <= 0 || d_state <= 0) return 0;
	return static_cast<size_t>(batch) * cdiv(seqlen, kTok) * dim * d_state * sizeof(float);
}

extern "C" int b200_selective_scan(int dtype, const b200_selective_scan_inputs* in, void* y, int64_t y_stride, float* final_state,
	float* checkpoints, void* workspace, size_t workspace_bytes, void* stream)
{
	int rc = selective_scan_check(dtype, in);
	if (rc != B200_OK) return rc;
	if (!y) return B200_ERR_NULL;
	if (y_stride < in->dim) return B200_ERR_BAD_SHAPE;
	if (!aligned16(in->initial_state) || !aligned16(final_state) || !aligned16(checkpoints)) return B200_ERR_MISALIGNED;
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	if (in->batch == 0) return B200_OK;
	if (in->seqlen == 0)
	{
		// no tokens: the state stays what it was
		const size_t bytes = static_cast<size_t>(in->batch) * in->dim * in->d_state * sizeof(float);
		if (final_state && in->initial_state && final_state != in->initial_state)
			B200_CUDA_TRY(cudaMemcpyAsync(final_state, in->initial_state, bytes, cudaMemcpyDeviceToDevice, st));
		else if (final_state && !in->initial_state) B200_CUDA_TRY(cudaMemsetAsync(final_state, 0, bytes, st));
		return B200_OK;
	}
	const Split sp = split_work(in->batch, in->seqlen, in->dim, in->ngroups, in->d_state, false);
	const size_t need = b200_selective_scan_workspace_bytes(in->batch, in->seqlen, in->dim, in->ngroups, in->d_state);
	if (need > 0 && (!workspace || workspace_bytes < need)) return B200_ERR_WORKSPACE;
	if (need > 0 && !aligned16(workspace)) return B200_ERR_MISALIGNED;
	float* ws = need > 0 ? static_cast<float*>(workspace) : nullptr;
	if (dtype == B200_F16) return scan<__half>(in, y, y_stride, final_state, checkpoints, ws, sp, st);
	return scan<float>(in, y, y_stride, final_state, checkpoints, ws, sp, st);
}

extern "C" int b200_selective_scan_update(int dtype, float* state, const void* x, int64_t x_stride, const void* dt, int64_t dt_stride,
	const float* A, int a_is_log, const void* B, int64_t B_stride, const void* C, int64_t C_stride, const float* D, const float* dt_bias,
	const void* z, int64_t z_stride, void* y, int64_t y_stride, int64_t batch, int64_t dim, int64_t ngroups, int64_t d_state,
	int dt_softplus, void* stream)
{
	b200_selective_scan_inputs in = { x, dt, B, C, z, x_stride, dt_stride, B_stride, C_stride, z_stride, A, D, dt_bias, nullptr, a_is_log,
		dt_softplus, batch, 1, dim, ngroups, d_state };
	const int rc = selective_scan_check(dtype, &in);
	if (rc != B200_OK) return rc;
	if (!state || !y) return B200_ERR_NULL;
	if (y_stride < dim) return B200_ERR_BAD_SHAPE;
	if (!aligned16(state)) return B200_ERR_MISALIGNED;
	if (batch == 0) return B200_OK;
	const Inputs p = selective_scan_params(&in, 0);
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	if (dtype == B200_F16) return scan_update<__half>(state, p, y, y_stride, batch, st);
	return scan_update<float>(state, p, y, y_stride, batch, st);
}
