// Gradient of the selective scan. With a_t = exp(delta_t A), u_t = delta_t x_t, s_t = sum_n C_t h_t + D x_t, y = s silu(z):
//   ds = dy silu(z);  dz = dy s silu'(z)
//   g_t = C_t ds_t + a_{t+1} g_{t+1}   (dfinal_state enters as the last a g)                    the adjoint of h_t, per channel and state
//   dC_t = sum_c ds_t h_t;  dB_t = sum_c g_t u_t                                                sums over the channels of a group
//   dx_t = D ds_t + delta_t sum_n g_t B_t;  ddelta_t = sum_n A (a_t g_t) h_{t-1} + x_t sum_n g_t B_t
//   ddt = ddelta softplus';  dA = sum_t delta_t (a_t g_t) h_{t-1};  dD = sum_t ds_t x_t;  dbias = sum_t ddt_t;  dinitial = a_0 g_0
// Threads load, lanes own states and warps own channels as in the forward kernel. A CTA walks its tokens backwards in tiles of 16: from the
// state the forward pass saved before the tile a warp runs the 16 tokens forward once, keeping every state in registers (16 x 4 per lane),
// then backwards for the adjoint; the decays are computed again on the way back, which costs less than the registers to keep them.
// 8192 x 4096 x 16 in f16: 1.04 ms. The 128 registers of a thread leave 14 - 16 warps per SM, which is what bounds it: 55% of the issue slots
// and 57% of the shared-memory pipe are used, a warp waits for fixed latencies 24%, at the two barriers of a tile 13%, for the multiply-add
// pipe 11% and for shared memory 10% of its time; HBM stands at 8%.
// dB and dC need a sum over channels: the lanes of a warp by exchanges, the warps of a CTA through shared memory, the CTAs as partial
// rows that a second kernel adds; dA, dD and dbias are summed over the tokens where they arise and leave one partial row per (batch
// entry, segment). No atomics anywhere.
// The exchanges halve what a lane holds instead of adding everything everywhere, and need no selects: the lanes of a channel hold their
// four states in an order that depends on the channel (state n0 + (i ^ p) in register i), so that the registers a lane sends are the
// same for all lanes and hold what its partner keeps. B and C are staged once per order.
// The activations of a tile are brought by asynchronous copies into slots that only the loading thread reads, one tile ahead; they
// stay there until the tile's gradients have been written.
#include <type_traits>

#include "column_reduce.cuh"
#include "selective_scan.cuh"

namespace b200 {

using namespace sscan;

struct BackwardArgs
{
	const void* dy;
	int64_t dys;
	const float *ckpt, *dfin;
	void *dx, *ddt, *dz;
	int64_t dxs, ddts, dzs;
	float* dinit;
	float* part_BC;   // [channel block of all groups][batch * seqlen][2][N] or null
	float* part_A;    // [batch * segments][dimN]
	float* part_D;    // [batch * segments][dimp]
	float* part_bias; // [batch * segments][dimp]
	int64_t dimp, dimN;  // dim and dim * N rounded up to 4
	float* seg_adj;   // [segments][batch][dim][N]: slot s = the adjoint that segment s hands to segment s - 1, from zero
	float* seg_dsum;  // [segments][batch][dim]
	int seg_tokens, nseg;
};

template <int LPC>
struct BackwardTile
{
	static constexpr int CW = warp_channels(LPC);
	static constexpr int EPT = CW < 2 ? 1 : CW / 2;  // channels of one token that a thread loads
	static constexpr int LPT = CW / EPT;             // threads per token and warp: two (one where a warp has one channel: half of them load)
	static constexpr int NP = LPC * kStates;
	static constexpr int ORDERS = CW >= 4 ? 4 : CW;  // orders of the four states, see Order
	static constexpr int PS = kTok + 1, DS = kTok + 1, RS = kTok + 4, YS = kTok + 4;  // padded rows of a channel (no bank conflicts)
};

// p of the lanes of warp channel cl: register i holds state n0 + (i ^ p). The first exchange is between channels that differ in bit X of
// cl and hands over registers 2 and 3, the second between those that differ in bit Y and hands over register 1; a third one, between
// channels that differ in bit 0, trades dB for dC. X and Y avoid bit 0 where they can: lanes i and i ^ 1 then read the same rows of B and C.
template <int LPC>
struct Order
{
	static constexpr int CW = warp_channels(LPC);
	static constexpr int X = CW >= 8 ? 1 : (CW == 4 ? 1 : 0), Y = CW >= 8 ? 2 : 0;
	static constexpr int lane_bit(int bit) { return bit == 0 ? 1 : LPC << bit; }  // of a channel bit (Lanes)
	static __device__ __forceinline__ int of(int cl) { return (CW > 1 ? ((cl >> X) & 1) << 1 : 0) | (CW > 2 ? (cl >> Y) & 1 : 0); }
};
__device__ __forceinline__ void permute(float* v, int p)
{
	const float a0 = p & 2 ? v[2] : v[0], a1 = p & 2 ? v[3] : v[1], a2 = p & 2 ? v[0] : v[2], a3 = p & 2 ? v[1] : v[3];
	v[0] = p & 1 ? a1 : a0;
	v[1] = p & 1 ? a0 : a1;
	v[2] = p & 1 ? a3 : a2;
	v[3] = p & 1 ? a2 : a3;
}

// Sums dB and dC of the lane's four states (in the order above) over the channels of the warp. On return the lane holds COUNT totals of
// each of ARRAYS arrays: of registers 0 .. COUNT - 1, in dB[] and dC[], or (ARRAYS = 1) in dB[0], which is dC's where bit 0 of cl is set.
template <int LPC>
struct ChannelSum
{
	static constexpr int CW = warp_channels(LPC);
	static constexpr int COUNT = CW >= 4 ? 1 : 4 / CW;
	static constexpr int ARRAYS = CW >= 8 ? 1 : 2;
	using O = Order<LPC>;
	static __device__ __forceinline__ f2 from(f2 v, int lane_bit)
	{
		const float2 a = unpack2(v);
		return pack2(__shfl_xor_sync(0xffffffffu, a.x, lane_bit), __shfl_xor_sync(0xffffffffu, a.y, lane_bit));
	}
	static __device__ __forceinline__ void run(f2 (&vB)[2], f2 (&vC)[2], int cl, float (&dB)[4], float (&dC)[4])
	{
		constexpr unsigned all = 0xffffffffu;
		if constexpr (CW >= 2)
		{
			vB[0] = add2(vB[0], from(vB[1], O::lane_bit(O::X)));
			vC[0] = add2(vC[0], from(vC[1], O::lane_bit(O::X)));
		}
		const float2 b0 = unpack2(vB[0]), b1 = unpack2(vB[1]), c0 = unpack2(vC[0]), c1 = unpack2(vC[1]);
		dB[0] = b0.x; dB[1] = b0.y; dB[2] = b1.x; dB[3] = b1.y;
		dC[0] = c0.x; dC[1] = c0.y; dC[2] = c1.x; dC[3] = c1.y;
		if constexpr (CW >= 4)
		{
			dB[0] += __shfl_xor_sync(all, dB[1], O::lane_bit(O::Y));
			dC[0] += __shfl_xor_sync(all, dC[1], O::lane_bit(O::Y));
		}
		if constexpr (CW >= 8)
		{
			const bool hi = cl & 1;
			const float send = hi ? dB[0] : dC[0];
			dB[0] = (hi ? dC[0] : dB[0]) + __shfl_xor_sync(all, send, 1);
#pragma unroll
			for (int bit = 3; (1 << bit) < CW; ++bit) dB[0] += __shfl_xor_sync(all, dB[0], O::lane_bit(bit));
		}
	}
};

// Bytes of shared memory of a CTA.
template <typename T, int LPC>
struct BackwardSmem
{
	using S = BackwardTile<LPC>;
	static constexpr int up16(int v) { return (v + 15) / 16 * 16; }
	static constexpr int P = S::CW * S::PS * 16;          // (delta, delta, u, u)
	static constexpr int DS = up16(S::CW * S::DS * 8);    // (ds, ds)
	static constexpr int R = up16(S::CW * S::RS * 8);     // (sum_n g B, sum_n A a g h)
	static constexpr int Y = up16(S::CW * S::YS * 4);     // sum_n C h
	static constexpr int ACC = 2 * S::EPT * 32 * 4;       // dD and dbias, per thread
	static constexpr int PAR = 2 * S::CW * 4;             // D and dt_bias
	static constexpr int FRAG = S::EPT * static_cast<int>(sizeof(T));  // bytes of one activation per thread
	static constexpr int RAW = 2 * 4 * 32 * (FRAG < 4 ? 4 : FRAG);     // two buffers of x, dt, z, dy
	static constexpr int RED = kTok * 2 * S::NP * 4;      // dB | dC
	// 16 bytes past a multiple of 128, which keeps apart the warps that neighbouring threads write to
	static constexpr int WARP = (P + DS + R + Y + ACC + RAW + RED + 111) / 128 * 128 + 16;
	// one order of B | C; 32 bytes more, so that the orders two apart, which half a warp reads together, lie in different banks
	static constexpr int BC = 2 * kTok * S::NP * 4 + (S::ORDERS > 1 ? 32 : 0);
	static constexpr int bytes(int warps) { return warps * (WARP + PAR) + S::ORDERS * BC; }
};

// MODE 1: what a segment does to the adjoint (for all segments but the first). MODE 0: the gradients.
template <typename T, int LPC, Access VEC, int MODE>
__global__ void __launch_bounds__(32 * kMaxWarps, 2) selective_scan_backward_kernel(const Inputs in, const BackwardArgs ar)
{
	using S = BackwardTile<LPC>;
	using M = BackwardSmem<T, LPC>;
	constexpr int CW = S::CW, EPT = S::EPT, LPT = S::LPT, NP = S::NP, PS = S::PS, DS = S::DS, RS = S::RS, YS = S::YS;
	constexpr int ROW = 2 * NP;
	extern __shared__ __align__(16) unsigned char smem[];
	const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	constexpr int AT_DS = M::P, AT_R = AT_DS + M::DS, AT_Y = AT_R + M::R, AT_ACC = AT_Y + M::Y, AT_RAW = AT_ACC + M::ACC, AT_RED = AT_RAW + M::RAW;
	constexpr int RAW1 = M::RAW / 8;                                           // one activation of one buffer
	unsigned char* own = smem + warp * M::WARP;
	float* s_acc = reinterpret_cast<float*>(own + AT_ACC);                     // [dD | dbias][EPT][lane], of the thread
	unsigned char* s_raw = own + AT_RAW;
	float* s_red = reinterpret_cast<float*>(own + AT_RED);                     // [kTok][dB | dC][NP]
	float* s_bc = reinterpret_cast<float*>(smem + warps * M::WARP);            // [ORDERS][B | C][kTok][NP]
	float* s_par = s_bc + S::ORDERS * (M::BC / 4);                             // [D | dt_bias][warps * CW]

	const int g = blockIdx.x / in.nbg;
	const int c0 = g * in.dpg + (blockIdx.x - g * in.nbg) * warps * CW;  // the CTA's first channel
	const int cend = (g + 1) * in.dpg;
	const int64_t b = blockIdx.y;
	const int seg = MODE == 1 ? blockIdx.z + 1 : blockIdx.z;
	const int64_t t_begin = static_cast<int64_t>(seg) * ar.seg_tokens;
	const int64_t t_end = t_begin + ar.seg_tokens < in.seqlen ? t_begin + ar.seg_tokens : in.seqlen;
	const int N = in.N;
	const bool vec4 = N % 4 == 0;

	// the thread's share of a tile: EPT channels from lc on of token lt, which another warp may own
	const int lt = threadIdx.x / (warps * LPT), lc = threadIdx.x % (warps * LPT) * EPT;
	const bool loads = lt < kTok;
	const int cn = loads ? cend - (c0 + lc) : 0;
	unsigned char* owner_s = smem + lc / CW * M::WARP;
	ulonglong2* t_p = reinterpret_cast<ulonglong2*>(owner_s) + lc % CW * PS + lt;
	f2* t_ds = reinterpret_cast<f2*>(owner_s + AT_DS) + lc % CW * DS + lt;
	const f2* t_r = reinterpret_cast<const f2*>(owner_s + AT_R) + lc % CW * RS + lt;
	const float* t_y = reinterpret_cast<const float*>(owner_s + AT_Y) + lc % CW * YS + lt;
	const float* t_skip = s_par + lc;
	const float* t_bias = s_par + warps * CW + lc;
	const int64_t tok0 = b * in.seqlen;
	const T* xp = static_cast<const T*>(in.x) + tok0 * in.xs + c0 + lc;
	const T* dp = static_cast<const T*>(in.dt) + tok0 * in.dts + c0 + lc;
	const T* zp = in.z ? static_cast<const T*>(in.z) + tok0 * in.zs + c0 + lc : nullptr;
	const T* yp = static_cast<const T*>(ar.dy) + tok0 * ar.dys + c0 + lc;
	const T* Bp = static_cast<const T*>(in.B) + tok0 * in.Bs + static_cast<int64_t>(g) * N;
	const T* Cp = static_cast<const T*>(in.C) + tok0 * in.Cs + static_cast<int64_t>(g) * N;
	for (int i = threadIdx.x; i < warps * CW; i += blockDim.x)
	{
		const bool ok = c0 + i < cend;
		s_par[i] = MODE == 0 && in.D && ok ? in.D[c0 + i] : 0.f;
		s_par[warps * CW + i] = in.bias && ok ? in.bias[c0 + i] : 0.f;
	}
	if (MODE == 0)
#pragma unroll
		for (int e = 0; e < 2 * EPT; ++e) s_acc[e * 32 + lane] = 0.f;
	__syncthreads();

	const int sub = Lanes<LPC>::sub(lane), cl = Lanes<LPC>::cl(lane), n0 = sub * kStates, c = c0 + warp * CW + cl;
	const int ord = Order<LPC>::of(cl);
	const bool mine = c < cend;
	const int64_t row = (b * in.dim + c) * N;
	const int64_t slots = static_cast<int64_t>(gridDim.y) * in.dim * N;
	auto load_ordered = [&](f2* h, const float* p) {
		float v[kStates];
		load_states(vec4, v, p, n0, N);
		permute(v, ord);
		h[0] = pack2(v[0], v[1]);
		h[1] = pack2(v[2], v[3]);
	};
	auto store_ordered = [&](const f2* h, float* p) {
		const float2 a = unpack2(h[0]), e = unpack2(h[1]);
		float v[kStates] = { a.x, a.y, e.x, e.y };
		permute(v, ord);  // its own inverse
		store_states(vec4, v, p, n0, N);
	};
	f2 a2[2] = { 0ull, 0ull }, carry[2] = { 0ull, 0ull }, aA[2] = { 0ull, 0ull };  // carry = a_{t+1} g_{t+1}
	float dsum = 0.f;
	if (mine)
	{
		float av[kStates];
		load_decay(av, in.A + static_cast<int64_t>(c) * N, in.a_is_log, n0, N);
		permute(av, ord);
		a2[0] = pack2(av[0], av[1]);
		a2[1] = pack2(av[2], av[3]);
		if (MODE == 0)
		{
			if (ar.dfin) load_ordered(carry, ar.dfin + row);
#pragma unroll 8  // the loads of eight segments at a time
			for (int q = ar.nseg - 1; q > seg; --q)
			{
				f2 add[2];
				load_ordered(add, ar.seg_adj + q * slots + row);
				const f2 ds = both(ar.seg_dsum[(static_cast<int64_t>(q) * gridDim.y + b) * in.dim + c]);
#pragma unroll
				for (int i = 0; i < 2; ++i) carry[i] = fma2(decay_2<true>(mul2(ds, a2[i])), carry[i], add[i]);
			}
		}
	}

	RowsBC<T, NP, kTok, 2> bc(threadIdx.x, blockDim.x);
	const bool vec_bc = in.vec_bc;
	float hn[kStates] = { 0.f, 0.f, 0.f, 0.f };  // the state before the next tile
	const int64_t nk = cdiv(in.seqlen, kTok);
	auto fetch = [&](int64_t t0, int buf, int pad) {
		const int64_t t = t0 + lt - pad;
		const int n = lt >= pad ? cn : 0;
		const int64_t tc = n > 0 ? t : t_begin;  // an address inside the tensor even where nothing is read
		unsigned char* r = s_raw + buf * 4 * RAW1;
		if (MODE == 0) raw_load<T, EPT, VEC>(r, xp + tc * in.xs, n, lane);
		raw_load<T, EPT, VEC>(r + RAW1, dp + tc * in.dts, n, lane);
		if (zp) raw_load<T, EPT, VEC>(r + 2 * RAW1, zp + tc * in.zs, n, lane);
		raw_load<T, EPT, VEC>(r + 3 * RAW1, yp + tc * ar.dys, n, lane);
		asm volatile("cp.async.commit_group;" ::: "memory");
		bc.fetch(vec_bc, in, Bp, Cp, t0 - pad, t_end, pad);
		if (MODE == 0 && mine) load_states(vec4, hn, ar.ckpt + ((b * nk + t0 / kTok) * in.dim + c) * N, n0, N);
	};
	// dB and dC of a finished tile: the warps in order, one partial row per CTA
	auto join_warps = [&](int64_t t0, int pad) {
		float* pr = ar.part_BC + (static_cast<int64_t>(blockIdx.x) * gridDim.y * in.seqlen + tok0 + t0 - pad) * 2 * N;
		for (int k = threadIdx.x * 4; k < kTok * ROW; k += blockDim.x * 4)
		{
			const int n = k % NP, t = k / ROW;
			if (n >= N || t < pad) continue;
			const unsigned char* r = smem + AT_RED + k * 4;  // of warp 0
			f2 s[2] = { 0ull, 0ull };
#pragma unroll
			for (int w = 0; w < kMaxWarps; ++w)
				if (w < warps)
				{
					const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(r + w * M::WARP);
					s[0] = add2(s[0], v.x);
					s[1] = add2(s[1], v.y);
				}
			store_states2(vec4, s, pr + (k / NP) * N, n, N);
		}
	};

	// A last tile that is not full has its empty places at the head (place lt is token t0 + lt - pad): the walk backwards meets its tokens
	// first, and what the empty places, whose steps are zero, make of NaN in A (exp(0 A)) comes after a token that did the same.
	const int64_t last = t_begin + (t_end - 1 - t_begin) / kTok * kTok;
	int pad = static_cast<int>(last + kTok - t_end);
	fetch(last, 0, pad);
	int buf = 0;
	for (int64_t t0 = last; t0 >= t_begin; t0 -= kTok, buf ^= 1, pad = 0)
	{
		const unsigned char* raw = s_raw + buf * 4 * RAW1;
		const bool tok = loads && lt >= pad;
		asm volatile("cp.async.wait_group 0;" ::: "memory");
		if (loads)
		{
			float dv[EPT], gv[EPT];
			raw_read<T, EPT>(raw + RAW1, dv, lane);
			raw_read<T, EPT>(raw + 3 * RAW1, gv, lane);
			if (zp)
			{
				float zv[EPT], sg[EPT];
				raw_read<T, EPT>(raw + 2 * RAW1, zv, lane);
				sigmoid_n<EPT, sizeof(T) == 4>(zv, sg);
#pragma unroll
				for (int e = 0; e < EPT; ++e) gv[e] *= zv[e] * sg[e];
			}
			float xv[EPT];
			if (MODE == 0) raw_read<T, EPT>(raw, xv, lane);
#pragma unroll
			for (int e = 0; e < EPT; ++e) dv[e] += t_bias[e];
			if (in.softplus) softplus_n<EPT>(dv);
#pragma unroll
			for (int e = 0; e < EPT; ++e)
			{
				const float dl = tok && e < cn ? dv[e] : 0.f;
				const float u = MODE == 0 ? dl * xv[e] : 0.f;
				t_p[e * PS] = make_ulonglong2(both(dl), both(u));
				t_ds[e * DS] = both(gv[e]);
			}
		}
		bc.template store_orders<S::ORDERS, M::BC / 4>(vec_bc, in, Bp, Cp, t0 - pad, t_end, pad, s_bc);
		const float* s_B = s_bc + (ord * S::ORDERS / 4) * (M::BC / 4);
		const float* s_C = s_B + kTok * NP;
		f2 hb[2];  // the state before this tile
		permute(hn, ord);
		hb[0] = pack2(hn[0], hn[1]);
		hb[1] = pack2(hn[2], hn[3]);
		__syncthreads();
		if (t0 > t_begin) fetch(t0 - kTok, buf ^ 1, 0);
		const ulonglong2* pp = reinterpret_cast<const ulonglong2*>(own) + cl * PS;
		const f2* pd = reinterpret_cast<const f2*>(own + AT_DS) + cl * DS;
		if constexpr (MODE == 1)
		{
#pragma unroll 4
			for (int t = kTok - 1; t >= 0; --t)
			{
				const ulonglong2 Cv = *reinterpret_cast<const ulonglong2*>(&s_C[t * NP + n0]);
				const f2 dl = pp[t].x, ds = pd[t];
				carry[0] = mul2(decay_2<true>(mul2(dl, a2[0])), fma2(Cv.x, ds, carry[0]));
				carry[1] = mul2(decay_2<true>(mul2(dl, a2[1])), fma2(Cv.y, ds, carry[1]));
				dsum += unpack2(dl).x;
			}
			__syncthreads();
		}
		else
		{
			float* s_y = reinterpret_cast<float*>(own + AT_Y) + cl * YS + TokenSum<LPC>::first(sub);
			f2* s_r = reinterpret_cast<f2*>(own + AT_R) + cl * RS + TokenSum<LPC>::first(sub);
			// as in the forward kernel, results wait in registers: stores to shared memory would hold back the next loads
			f2 h[kTok][2];
			float tot[kTok / 4][TokenSum<LPC>::COUNT];
#pragma unroll
			for (int t4 = 0; t4 < kTok; t4 += 4)
			{
				float acc[4];
#pragma unroll
				for (int j = 0; j < 4; ++j)
				{
					const int t = t4 + j;
					const ulonglong2 p = pp[t];
					const ulonglong2 Bv = *reinterpret_cast<const ulonglong2*>(&s_B[t * NP + n0]);
					const ulonglong2 Cv = *reinterpret_cast<const ulonglong2*>(&s_C[t * NP + n0]);
					h[t][0] = fma2(decay_2<sizeof(T) == 4>(mul2(p.x, a2[0])), t == 0 ? hb[0] : h[t - 1][0], mul2(p.y, Bv.x));
					h[t][1] = fma2(decay_2<sizeof(T) == 4>(mul2(p.x, a2[1])), t == 0 ? hb[1] : h[t - 1][1], mul2(p.y, Bv.y));
					acc[j] = sum2(fma2(h[t][1], Cv.y, mul2(h[t][0], Cv.x)));
				}
				TokenSum<LPC>::run(acc, sub, tot[t4 / 4]);
			}
			if (TokenSum<LPC>::owner(sub))
#pragma unroll
				for (int i = 0; i < kTok / 4; ++i)
#pragma unroll
					for (int j = 0; j < TokenSum<LPC>::COUNT; ++j) s_y[i * 4 + j] = tot[i][j];
			// where the lane's totals go: state n0 + (i ^ ord) of array 0 (dB) or 1 (dC)
			float* red = s_red + n0 + (ChannelSum<LPC>::ARRAYS == 1 && (cl & 1) ? NP : 0);
			const bool owner = CW <= 8 || cl < 8;
			struct Step
			{
				ulonglong2 p, B, C;
				f2 ds;
			};
			auto load_step = [&](int t) {
				return Step{ pp[t], *reinterpret_cast<const ulonglong2*>(&s_B[t * NP + n0]), *reinterpret_cast<const ulonglong2*>(&s_C[t * NP + n0]), pd[t] };
			};
			f2 tile_A[2] = { 0ull, 0ull };  // the tile's part of dA: the running sum over all tokens takes 16 terms at a time
			Step next = load_step(kTok - 1);
#pragma unroll
			for (int t4 = kTok - 4; t4 >= 0; t4 -= 4)
			{
				float gB[4], gA[4];
#pragma unroll
				for (int j = 3; j >= 0; --j)
				{
					const int t = t4 + j;
					const Step s = next;
					if (t > 0) next = load_step(t - 1);
					const f2 g0 = fma2(s.C.x, s.ds, carry[0]), g1 = fma2(s.C.y, s.ds, carry[1]);
					gB[j] = sum2(fma2(g1, s.B.y, mul2(g0, s.B.x)));
					carry[0] = mul2(decay_2<true>(mul2(s.p.x, a2[0])), g0);
					carry[1] = mul2(decay_2<true>(mul2(s.p.x, a2[1])), g1);
					const f2 q0 = mul2(carry[0], t == 0 ? hb[0] : h[t - 1][0]);
					const f2 q1 = mul2(carry[1], t == 0 ? hb[1] : h[t - 1][1]);
					gA[j] = sum2(fma2(a2[1], q1, mul2(a2[0], q0)));
					tile_A[0] = fma2(s.p.x, q0, tile_A[0]);
					tile_A[1] = fma2(s.p.x, q1, tile_A[1]);
					f2 pB[2] = { mul2(g0, s.p.y), mul2(g1, s.p.y) }, pC[2] = { mul2(h[t][0], s.ds), mul2(h[t][1], s.ds) };
					float vB[4], vC[4];
					ChannelSum<LPC>::run(pB, pC, cl, vB, vC);
					if (owner)
#pragma unroll
						for (int i = 0; i < ChannelSum<LPC>::COUNT; ++i)
						{
							red[t * ROW + (i ^ ord)] = vB[i];
							if (ChannelSum<LPC>::ARRAYS == 2) red[t * ROW + NP + (i ^ ord)] = vC[i];
						}
				}
				float tB[TokenSum<LPC>::COUNT], tA[TokenSum<LPC>::COUNT];
				TokenSum<LPC>::run(gB, sub, tB);
				TokenSum<LPC>::run(gA, sub, tA);
				if (TokenSum<LPC>::owner(sub))
#pragma unroll
					for (int i = 0; i < TokenSum<LPC>::COUNT; ++i) s_r[t4 + i] = pack2(tB[i], tA[i]);
			}
			aA[0] = add2(aA[0], tile_A[0]);
			aA[1] = add2(aA[1], tile_A[1]);
			__syncthreads();
			if (ar.part_BC) join_warps(t0, pad);
			if (tok)
			{
				const int64_t t = tok0 + t0 + lt - pad;
				float xv[EPT], dv[EPT], gv[EPT], zv[EPT], ox[EPT], od[EPT], ds[EPT];
				raw_read<T, EPT>(raw, xv, lane);
				raw_read<T, EPT>(raw + RAW1, dv, lane);
				raw_read<T, EPT>(raw + 3 * RAW1, gv, lane);
				if (zp)
				{
					float sg[EPT];
					raw_read<T, EPT>(raw + 2 * RAW1, zv, lane);
					sigmoid_n<EPT, sizeof(T) == 4>(zv, sg);
#pragma unroll
					for (int e = 0; e < EPT; ++e)
					{
						ds[e] = gv[e] * zv[e] * sg[e];
						zv[e] = gv[e] * (t_y[e * YS] + t_skip[e] * xv[e]) * (sg[e] * (1.f + zv[e] * (1.f - sg[e])));
					}
					if (ar.dz) store_frag<T, EPT, VEC>(zv, static_cast<T*>(ar.dz) + t * ar.dzs + c0 + lc, cn);
				}
				else
#pragma unroll
					for (int e = 0; e < EPT; ++e) ds[e] = gv[e];
#pragma unroll
				for (int e = 0; e < EPT; ++e) dv[e] += t_bias[e];
				if (in.softplus) sigmoid_n<EPT, true>(dv, dv);
#pragma unroll
				for (int e = 0; e < EPT; ++e)
				{
					const float2 s = unpack2(t_r[e * RS]);
					const float dl = unpack2(t_p[e * PS].x).x;
					ox[e] = t_skip[e] * ds[e] + dl * s.x;
					// A step that softplus left at zero has no gradient. The sum over A does not enter then: where A is the type's lowest value
					// it overflows, and softplus' = 0 would turn that into NaN.
					od[e] = (in.softplus && dl == 0.f ? 0.f : s.y * (1.f / kLog2e)) + xv[e] * s.x;
					if (in.softplus) od[e] *= dv[e];
					s_acc[e * 32 + lane] += ds[e] * xv[e];
					s_acc[(EPT + e) * 32 + lane] += od[e];
				}
				if (ar.dx) store_frag<T, EPT, VEC>(ox, static_cast<T*>(ar.dx) + t * ar.dxs + c0 + lc, cn);
				if (ar.ddt) store_frag<T, EPT, VEC>(od, static_cast<T*>(ar.ddt) + t * ar.ddts + c0 + lc, cn);
			}
		}
	}
	if constexpr (MODE == 1)
	{
		if (!mine) return;
		store_ordered(carry, ar.seg_adj + seg * slots + row);
		if (sub == 0) ar.seg_dsum[(static_cast<int64_t>(seg) * gridDim.y + b) * in.dim + c] = dsum;
	}
	else
	{
		const int64_t pr = b * ar.nseg + seg;  // partial row
		if (mine)
		{
			if (ar.dinit && seg == 0) store_ordered(carry, ar.dinit + row);
			if (ar.part_A)
			{
				if (in.a_is_log)  // with respect to A_log: A = -exp(A_log), dA/dA_log = A
#pragma unroll
					for (int i = 0; i < 2; ++i) aA[i] = mul2(aA[i], mul2(a2[i], both(1.f / kLog2e)));
				store_ordered(aA, ar.part_A + pr * ar.dimN + static_cast<int64_t>(c) * N);
			}
		}
		// the 16 threads that loaded a channel hold the sums over their tokens of every tile
		__syncthreads();
		for (int i = threadIdx.x; i < warps * CW; i += blockDim.x)
		{
			if (c0 + i >= cend) continue;
			float sD = 0.f, sb = 0.f;
#pragma unroll
			for (int t = 0; t < kTok; ++t)
			{
				const int th = t * warps * LPT + i / EPT;
				const float* acc = reinterpret_cast<const float*>(smem + (th >> 5) * M::WARP + AT_ACC) + (th & 31);
				sD += acc[i % EPT * 32];
				sb += acc[(EPT + i % EPT) * 32];
			}
			if (ar.part_D) ar.part_D[pr * ar.dimp + c0 + i] = sD;
			if (ar.part_bias) ar.part_bias[pr * ar.dimp + c0 + i] = sb;
		}
	}
}

// dB and dC: adds the channel blocks of a group in order. One thread per (token, array, group, state).
template <typename T>
__global__ void __launch_bounds__(256) selective_scan_bc_kernel(const float* __restrict__ part, T* __restrict__ dB, int64_t dBs,
	T* __restrict__ dC, int64_t dCs, int64_t tokens, int N, int nbg)
{
	const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
	const int g = blockIdx.y;
	if (i >= tokens * 2 * N) return;
	const int64_t tokk = i / (2 * N);
	const int r = static_cast<int>(i - tokk * 2 * N);
	float s = 0.f;
	const float* p = part + static_cast<int64_t>(g) * nbg * tokens * 2 * N + i;
#pragma unroll 8
	for (int k = 0; k < nbg; ++k) s += p[static_cast<int64_t>(k) * tokens * 2 * N];
	T* out = r < N ? dB : dC;
	if (out) stf(out + tokk * (r < N ? dBs : dCs) + static_cast<int64_t>(g) * N + (r < N ? r : r - N), s);
}

// ---- host ------------------------------------------------------------------------------------------------------------

namespace sscan {
int backward_smem_bytes(int lpc, int warps)
{
	switch (lpc)
	{
	case 1: return BackwardSmem<__half, 1>::bytes(warps);
	case 2: return BackwardSmem<__half, 2>::bytes(warps);
	case 4: return BackwardSmem<__half, 4>::bytes(warps);
	case 8: return BackwardSmem<__half, 8>::bytes(warps);
	case 16: return BackwardSmem<__half, 16>::bytes(warps);
	default: return BackwardSmem<__half, 32>::bytes(warps);
	}
}
}  // namespace sscan

struct BackwardPlan
{
	Split sp;
	int nblocks;
	size_t bc, pa, pd, adj, dsum;  // floats of each part of the workspace, multiples of 4
	int64_t dimp, dimN;
	size_t total() const { return bc + pa + 2 * pd + adj + dsum; }
};

static BackwardPlan backward_plan(int64_t batch, int64_t seqlen, int64_t dim, int64_t ngroups, int64_t N)
{
	auto up4 = [](int64_t v) { return static_cast<size_t>(cdiv(v, 4) * 4); };
	BackwardPlan p;
	p.sp = split_work(batch, seqlen, dim, ngroups, N, true);
	p.nblocks = static_cast<int>(ngroups * p.sp.nbg);
	p.dimp = cdiv(dim, 4) * 4;
	p.dimN = cdiv(dim * N, 4) * 4;
	p.bc = up4(static_cast<int64_t>(p.nblocks) * batch * seqlen * 2 * N);
	p.pa = static_cast<size_t>(batch) * p.sp.nseg * p.dimN;
	p.pd = static_cast<size_t>(batch) * p.sp.nseg * p.dimp;
	p.adj = p.sp.nseg > 1 ? up4(static_cast<int64_t>(p.sp.nseg) * batch * dim * N) : 0;
	p.dsum = p.sp.nseg > 1 ? up4(static_cast<int64_t>(p.sp.nseg) * batch * dim) : 0;
	return p;
}

template <typename T, int LPC, Access VEC, int MODE>
static int launch_backward_kernel(const Split& sp, const dim3& g, const Inputs& p, const BackwardArgs& ar, cudaStream_t st)
{
	using M = BackwardSmem<T, LPC>;
	static_assert(M::bytes(max_warps(LPC)) <= 232448, "shared memory of a CTA");
	static bool done[64];
	B200_CUDA_TRY(allow_dynamic_smem(selective_scan_backward_kernel<T, LPC, VEC, MODE>, M::bytes(max_warps(LPC)), done));
	selective_scan_backward_kernel<T, LPC, VEC, MODE><<<g, 32 * sp.warps, M::bytes(sp.warps), st>>>(p, ar);
	B200_LAUNCH_CHECK();
	return B200_OK;
}

template <typename T, int LPC>
static int launch_backward(const b200_selective_scan_inputs* in, const Split& sp, const BackwardArgs& ar, cudaStream_t st)
{
	constexpr int EPT = BackwardTile<LPC>::EPT;
	Inputs p = selective_scan_params(in, sp.nbg);
	p.vec_bc = RowsBC<T, BackwardTile<LPC>::NP, kTok, 2>::aligned(in);
	auto al = [](const void* q, int64_t stride) { return frag_aligned<T, EPT>(q, stride); };
	const bool vec = p.dpg % EPT == 0 && al(p.x, p.xs) && al(p.dt, p.dts) && al(p.z, p.zs) && al(ar.dy, ar.dys) && al(ar.dx, ar.dxs) &&
		al(ar.ddt, ar.ddts) && al(ar.dz, ar.dzs);
	const bool words = sizeof(T) == 2 && p.dpg % 2 == 0 && word_aligned(p.x, p.xs) && word_aligned(p.dt, p.dts) && word_aligned(p.z, p.zs) &&
		word_aligned(ar.dy, ar.dys) && word_aligned(ar.dx, ar.dxs) && word_aligned(ar.ddt, ar.ddts) && word_aligned(ar.dz, ar.dzs);
	const dim3 g(static_cast<unsigned>(in->ngroups * p.nbg), static_cast<unsigned>(in->batch), static_cast<unsigned>(sp.nseg));
	auto run = [&](auto access) {
		constexpr Access VEC = decltype(access)::value;
		if (sp.nseg > 1)
		{
			const dim3 g1(g.x, g.y, g.z - 1);
			const int rc = launch_backward_kernel<T, LPC, VEC, 1>(sp, g1, p, ar, st);
			if (rc != B200_OK) return rc;
		}
		return launch_backward_kernel<T, LPC, VEC, 0>(sp, g, p, ar, st);
	};
	if (vec) return run(std::integral_constant<Access, kVectors>{});
	if constexpr (sizeof(T) == 2)
		if (words) return run(std::integral_constant<Access, kWords>{});
	return run(std::integral_constant<Access, kSingle>{});
}

template <typename T>
static int scan_backward(const b200_selective_scan_inputs* in, const Split& sp, const BackwardArgs& ar, const b200_selective_scan_grads* gr, cudaStream_t st)
{
	int rc;
	switch (lanes_per_channel(in->d_state))
	{
	case 1: rc = launch_backward<T, 1>(in, sp, ar, st); break;
	case 2: rc = launch_backward<T, 2>(in, sp, ar, st); break;
	case 4: rc = launch_backward<T, 4>(in, sp, ar, st); break;
	case 8: rc = launch_backward<T, 8>(in, sp, ar, st); break;
	case 16: rc = launch_backward<T, 16>(in, sp, ar, st); break;
	default: rc = launch_backward<T, 32>(in, sp, ar, st); break;
	}
	if (rc != B200_OK) return rc;
	if (ar.part_BC)
	{
		const int64_t tokens = in->batch * in->seqlen;
		const int N = static_cast<int>(in->d_state);
		const int64_t blocks = cdiv(tokens * 2 * N, 256);
		if (blocks > 0x7fffffffLL) return B200_ERR_UNSUPPORTED;
		selective_scan_bc_kernel<T><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(in->ngroups)), 256, 0, st>>>(ar.part_BC,
			static_cast<T*>(gr->dB), gr->dB_stride, static_cast<T*>(gr->dC), gr->dC_stride, tokens, N, sp.nbg);
		B200_LAUNCH_CHECK();
	}
	ReduceJobs jobs = {};
	int n = 0;
	if (gr->dA) jobs.j[n++] = { ar.part_A, ar.dimN, in->dim * in->d_state, gr->dA, 1 };
	if (gr->dD) jobs.j[n++] = { ar.part_D, ar.dimp, in->dim, gr->dD, 1 };
	if (gr->ddt_bias) jobs.j[n++] = { ar.part_bias, ar.dimp, in->dim, gr->ddt_bias, 1 };
	return n > 0 ? column_reduce(jobs, n, static_cast<int>(in->batch * sp.nseg), st) : B200_OK;
}

}  // namespace b200

using namespace b200;

extern "C" size_t b200_selective_scan_backward_workspace_bytes(int64_t batch, int64_t seqlen, int64_t dim, int64_t ngroups, int64_t d_state)
{
	if (batch <= 0 || seqlen <= 0 || dim <= 0 || ngroups <= 0 || d_state <= 0 || dim % ngroups != 0 || d_state > kMaxState) return 0;
	return backward_plan(batch, seqlen, dim, ngroups, d_state).total() * sizeof(float);
}

extern "C" int b200_selective_scan_backward(int dtype, const b200_selective_scan_inputs* in, const float* checkpoints, const void* dy,
	int64_t dy_stride, const float* dfinal_state, const b200_selective_scan_grads* gr, void* workspace, size_t workspace_bytes, void* stream)
{
	const int rc = selective_scan_check(dtype, in);
	if (rc != B200_OK) return rc;
	if (!dy || !gr) return B200_ERR_NULL;
	if (in->seqlen > 0 && in->batch > 0 && !checkpoints) return B200_ERR_NULL;
	if ((gr->dz && !in->z) || (gr->dD && !in->D) || (gr->ddt_bias && !in->dt_bias)) return B200_ERR_NULL;
	const int64_t gn = in->ngroups * in->d_state;
	if (dy_stride < in->dim || (gr->dx && gr->dx_stride < in->dim) || (gr->ddt && gr->ddt_stride < in->dim) || (gr->dz && gr->dz_stride < in->dim) ||
		(gr->dB && gr->dB_stride < gn) || (gr->dC && gr->dC_stride < gn))
		return B200_ERR_BAD_SHAPE;
	if (!aligned16(checkpoints) || !aligned16(dfinal_state) || !aligned16(gr->dinitial_state)) return B200_ERR_MISALIGNED;
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	if (in->batch == 0 || in->seqlen == 0)
	{
		// sums over no tokens; the state's gradient passes through
		const size_t dim = static_cast<size_t>(in->dim), state = dim * in->d_state * sizeof(float);
		if (gr->dA) B200_CUDA_TRY(cudaMemsetAsync(gr->dA, 0, state, st));
		if (gr->dD) B200_CUDA_TRY(cudaMemsetAsync(gr->dD, 0, dim * sizeof(float), st));
		if (gr->ddt_bias) B200_CUDA_TRY(cudaMemsetAsync(gr->ddt_bias, 0, dim * sizeof(float), st));
		if (gr->dinitial_state && in->batch > 0)
		{
			if (dfinal_state) B200_CUDA_TRY(cudaMemcpyAsync(gr->dinitial_state, dfinal_state, in->batch * state, cudaMemcpyDeviceToDevice, st));
			else B200_CUDA_TRY(cudaMemsetAsync(gr->dinitial_state, 0, in->batch * state, st));
		}
		return B200_OK;
	}
	const BackwardPlan p = backward_plan(in->batch, in->seqlen, in->dim, in->ngroups, in->d_state);
	if (!workspace || workspace_bytes < p.total() * sizeof(float)) return B200_ERR_WORKSPACE;
	if (!aligned16(workspace)) return B200_ERR_MISALIGNED;
	float* w = static_cast<float*>(workspace);
	BackwardArgs ar = {};
	ar.dy = dy; ar.dys = dy_stride;
	ar.ckpt = checkpoints; ar.dfin = dfinal_state;
	ar.dx = gr->dx; ar.ddt = gr->ddt; ar.dz = gr->dz;
	ar.dxs = gr->dx_stride; ar.ddts = gr->ddt_stride; ar.dzs = gr->dz_stride;
	ar.dinit = gr->dinitial_state;
	ar.part_BC = gr->dB || gr->dC ? w : nullptr;
	ar.part_A = gr->dA ? w + p.bc : nullptr;
	ar.part_D = gr->dD ? w + p.bc + p.pa : nullptr;
	ar.part_bias = gr->ddt_bias ? w + p.bc + p.pa + p.pd : nullptr;
	ar.dimp = p.dimp; ar.dimN = p.dimN;
	ar.seg_adj = p.sp.nseg > 1 ? w + p.bc + p.pa + 2 * p.pd : nullptr;
	ar.seg_dsum = p.sp.nseg > 1 ? ar.seg_adj + p.adj : nullptr;
	ar.seg_tokens = p.sp.seg_tokens; ar.nseg = p.sp.nseg;
	if (p.sp.nseg > 1 && dfinal_state && dfinal_state == gr->dinitial_state)
	{
		// in place: the first segment may write its gradient before a later one has read; slot 0 of the adjoints is free
		B200_CUDA_TRY(cudaMemcpyAsync(ar.seg_adj, dfinal_state, static_cast<size_t>(in->batch * in->dim * in->d_state) * sizeof(float),
			cudaMemcpyDeviceToDevice, st));
		ar.dfin = ar.seg_adj;
	}
	if (dtype == B200_F16) return scan_backward<__half>(in, p.sp, ar, gr, st);
	return scan_backward<float>(in, p.sp, ar, gr, st);
}
