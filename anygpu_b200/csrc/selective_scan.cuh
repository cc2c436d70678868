// Shared parts of the selective scan kernels (forward, single token, backward).
#pragma once
#include "packed.cuh"

namespace b200 {
namespace sscan {

constexpr int kStates = 4;    // states of one channel that a lane owns: two pairs for the packed fp32 instructions
constexpr int kTok = 16;      // tokens between two saved states, from which the backward pass recomputes
constexpr int kMaxState = 32 * kStates;
constexpr int kMaxWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = static_cast<float>(1.4426950408889634 - static_cast<double>(kLog2e));  // log2(e) = kLog2e + kLog2eLow

// Lanes that share a channel of n states: the smallest power of two whose lanes hold them all.
inline int lanes_per_channel(int64_t n)
{
	int l = 1;
	while (l * kStates < n) l *= 2;
	return l;
}
// Channels of a warp.
constexpr int warp_channels(int lpc) { return 32 / lpc; }
// Warps of a CTA at most (32 channels per warp fill the backward kernel's shared memory sooner).
constexpr int max_warps(int lpc) { return lpc == 1 ? 4 : kMaxWarps; }

struct Inputs
{
	const void *x, *dt, *B, *C, *z;
	int64_t xs, dts, Bs, Cs, zs;
	const float *A, *D, *bias, *init;
	int a_is_log, softplus;
	int64_t seqlen;
	int dim, N, dpg /* channels per group */, nbg /* channel blocks (CTAs) per group */;
	int vec_bc;  // RowsBC::aligned
};

__device__ __forceinline__ float exp2_approx(float v)
{
	float r;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
	return r;
}
__device__ __forceinline__ f2 exp2_2(f2 a)
{
	const float2 v = unpack2(a);
	return pack2(exp2_approx(v.x), exp2_approx(v.y));
}
// 2^(n + f) of a pair: f in [-1/2, 1/2] up to rounding, t = 1.5 * 2^23 + n, which holds the integer n in its low bits. 2^f by its minimax
// polynomial of degree 6 with constant term 1 (relative error 2^-28.9, and exact at 0, where the decays of slow states lie), times the
// float whose exponent field is n + 127, n in [-127, 128]. (An integer addition of n to the polynomial's exponent would save that
// multiplication, but turns NaN into a number.)
__device__ __forceinline__ f2 pow2_split(f2 t, f2 f)
{
	f2 p = both(1.535336179e-04f);
	p = fma2(p, f, both(1.339887446e-03f));
	p = fma2(p, f, both(9.618437358e-03f));
	p = fma2(p, f, both(5.550332471e-02f));
	p = fma2(p, f, both(2.402264791e-01f));
	p = fma2(p, f, both(6.931472029e-01f));
	p = fma2(p, f, both(1.f));
	const float2 n = unpack2(t);
	return mul2(p, pack2(__int_as_float((__float_as_int(n.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(n.y) << 23) + 0x3f800000)));
}
// NaN stays NaN.
template <bool LOW_ONLY = false>
__device__ __forceinline__ f2 clamp_2(f2 x, float lo, float hi)
{
	float2 v = unpack2(x);
	asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(lo));
	asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(lo));
	if constexpr (!LOW_ONLY)
	{
		asm("min.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(hi));
		asm("min.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(hi));
	}
	return pack2(v.x, v.y);
}
// 2^x of a pair to half a step of fp32, without the exponential unit: x = n + f, n the nearest integer (added and taken away with
// 1.5 * 2^23). Below x = -126.5 the exponent field is 0 and the result zero: a decay that forgets the state leaves nothing of it for A,
// which may be as large as floats go, to magnify in the gradients. From x = 127.5 on the result is infinite, NaN stays NaN.
__device__ __forceinline__ f2 exp2_poly_2(f2 x)
{
	const f2 c = clamp_2(x, -127.f, 128.f);
	const f2 t = add2(c, both(12582912.f));
	return pow2_split(t, add2(c, fma2(t, both(-1.f), both(12582912.f))));
}
// e^v of a pair to two half steps (2^-24) of fp32. v log2(e) rounded once would be off by |v| half steps of the result; here the integer part is taken
// from it and the fraction is v log2(e) - n in multiply-adds, which round once, with log2(e) in two floats. Zero below v = -87.7, infinite from
// 88.4 on, NaN stays NaN.
template <bool NEGATIVE = false /* v <= 0 */>
__device__ __forceinline__ f2 exp_2(f2 v)
{
	const f2 c = clamp_2<NEGATIVE>(v, -88.1f, 88.6f);  // times log2(e): -127.1, 127.8
	const f2 t = fma2(c, both(kLog2e), both(12582912.f));
	f2 f = fma2(c, both(kLog2e), fma2(t, both(-1.f), both(12582912.f)));
	f = fma2(c, both(kLog2eLow), f);
	return pow2_split(t, f);
}
// The decays of one token. The exponential unit's 2^-22 adds up over a long memory: with it everywhere dA is off by 1.8e-6 and
// final_state by 4.7e-7 (8192 x 4096 x 16, f16 activations), with the polynomial everywhere by 3.4e-7 and 1.2e-7, at 406 instead of 230 us
// forward and 1644 instead of 1275 per training step. So fp32 calls, whose results show it, take the polynomial everywhere; f16 calls take it
// in the adjoint recurrence (dA 9.5e-7; the training step 1275 instead of 1116 us), between segments and for single tokens (64 x 5120 x 16:
// 15.7 us instead of 14.4).
template <bool EXACT>
__device__ __forceinline__ f2 decay_2(f2 x)
{
	if constexpr (EXACT) return exp2_poly_2(x);
	else return exp2_2(x);
}
__device__ __forceinline__ float rcp_approx(float v)
{
	float r;
	asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
	return r;
}

__device__ __forceinline__ f2 rcp_2(f2 a)
{
	const float2 v = unpack2(a);
	return pack2(rcp_approx(v.x), rcp_approx(v.y));
}

// softplus(v) = max(v, 0) + log1p(w), w = exp(-|v|) <= 1, and log1p(w) = 2 artanh(s), s = w / (2 + w) <= 1/3, by the series of artanh
// through s^13 (the next term is below 2^-25 of the sum). Relative accuracy holds down to the smallest steps, which a logarithm of
// 1 + w would lose. NaN stays NaN.
__device__ __forceinline__ f2 softplus_2(f2 v)
{
	const float2 a = unpack2(v);
	const f2 w = exp_2<true>(pack2(-fabsf(a.x), -fabsf(a.y)));
	const f2 s = mul2(w, rcp_2(add2(w, both(2.f))));
	const f2 q = mul2(s, s);
	f2 p = both(2.f / 13.f);
	p = fma2(p, q, both(2.f / 11.f));
	p = fma2(p, q, both(2.f / 9.f));
	p = fma2(p, q, both(2.f / 7.f));
	p = fma2(p, q, both(2.f / 5.f));
	p = fma2(p, q, both(2.f / 3.f));
	p = fma2(p, q, both(2.f));
	return fma2(p, s, pack2(a.x > 0.f ? a.x : 0.f, a.y > 0.f ? a.y : 0.f));
}
// 1 / (1 + exp(-v)). EXACT (fp32 calls, and softplus' everywhere, which ddt_bias sums in fp32): e^-v to two half steps. Else through the exponential
// unit, off by |v| half steps for the rounding of v log2(e): the gate of f16 calls, whose results are rounded by 2^13 of them. (With it everywhere
// the step sizes were off by 1.7e-7 rms instead of 6.8e-8 and those at v = -60 by 56 u. It costs the f16 training step of 4 x 2048 x 4096 x 16 1250 ->
// 1275 us, the prompt 228 -> 230; with the gates too 1304 and 231. fp32: prompt 438 -> 429, training step of 4 x 1024 835 -> 860.)
template <bool EXACT>
__device__ __forceinline__ f2 sigmoid_2(f2 v)
{
	const f2 e = EXACT ? exp_2(mul2(v, both(-1.f))) : exp2_2(mul2(v, both(-kLog2e)));
	return rcp_2(add2(e, both(1.f)));
}
// The same functions over an even or odd number of values.
template <int E>
__device__ __forceinline__ void softplus_n(float* v)
{
#pragma unroll
	for (int e = 0; e < E; e += 2)
	{
		const float2 r = unpack2(softplus_2(pack2(v[e], v[e + 1 < E ? e + 1 : e])));
		v[e] = r.x;
		if (e + 1 < E) v[e + 1] = r.y;
	}
}
template <int E, bool EXACT>
__device__ __forceinline__ void sigmoid_n(const float* v, float* o)
{
#pragma unroll
	for (int e = 0; e < E; e += 2)
	{
		const float2 r = unpack2(sigmoid_2<EXACT>(pack2(v[e], v[e + 1 < E ? e + 1 : e])));
		o[e] = r.x;
		if (e + 1 < E) o[e + 1] = r.y;
	}
}

template <typename T, int EPT>
struct alignas(16) Frag
{
	T v[EPT];
};

// How a thread reads and writes EPT consecutive channels of one token: single elements; four bytes at a time (f16 rows off 16 bytes but on 4,
// channels of a group even); 16 bytes (or the EPT elements) at a time. 4 x 1024 tokens x 16 states, f16: 2049 channels one by one 110 us,
// 2050 by four bytes 72 (one by one 109), 2048 67; fp32 elements one by one 133, asynchronously 141.
enum Access { kSingle, kWords, kVectors };

// Missing channels read zero and are not written.
template <typename T, int EPT>
__device__ __forceinline__ void load_frag(Frag<T, EPT>& f, const T* p, int n)
{
#pragma unroll
	for (int e = 0; e < EPT; ++e) f.v[e] = e < n ? p[e] : Cvt<T>::from_f32(0.f);
}
template <typename T, int EPT, Access VEC>
__device__ __forceinline__ void store_frag(const float* o, T* p, int n)
{
	if constexpr (VEC == kVectors)
	{
		if (n <= 0) return;
		constexpr int BYTES = EPT * sizeof(T) < 16 ? EPT * sizeof(T) : 16;
		constexpr int PV = BYTES / sizeof(T);
#pragma unroll
		for (int i = 0; i < EPT / PV; ++i)
		{
			Pack<T, PV> q;
			q.pack(o + i * PV);
			q.store(p + i * PV);
		}
	}
	else if constexpr (VEC == kWords && EPT % 2 == 0)
	{
#pragma unroll
		for (int e = 0; e < EPT; e += 2)
			if (e < n) *reinterpret_cast<__half2*>(p + e) = __floats2half2_rn(o[e], o[e + 1]);
	}
	else
	{
#pragma unroll
		for (int e = 0; e < EPT; ++e)
			if (e < n) stf(p + e, o[e]);
	}
}
template <typename T, int EPT>
__device__ __forceinline__ void frag_f32(const Frag<T, EPT>& f, float* o)
{
	if constexpr (sizeof(T) == 2 && EPT % 2 == 0)
	{
#pragma unroll
		for (int e = 0; e < EPT; e += 2)
		{
			const float2 t = __half22float2(*reinterpret_cast<const __half2*>(f.v + e));
			o[e] = t.x;
			o[e + 1] = t.y;
		}
	}
	else
	{
#pragma unroll
		for (int e = 0; e < EPT; ++e) o[e] = Cvt<T>::to_f32(f.v[e]);
	}
}
// Whether a tensor's rows allow kVectors: EPT channels at a time from channel offsets that are multiples of EPT.
template <typename T, int EPT>
inline bool frag_aligned(const void* p, int64_t stride)
{
	constexpr int BYTES = EPT * sizeof(T) < 16 ? EPT * sizeof(T) : 16;
	return !p || (reinterpret_cast<uintptr_t>(p) % BYTES == 0 && stride * static_cast<int64_t>(sizeof(T)) % BYTES == 0);
}

// The same for kWords (f16).
inline bool word_aligned(const void* p, int64_t stride) { return !p || (reinterpret_cast<uintptr_t>(p) % 4 == 0 && stride % 2 == 0); }

// One activation of one thread: EPT elements into the thread's slot, asynchronously where the rows allow it. chunk = 16 bytes (or the
// whole fragment); the chunks of a warp's lanes lie side by side.
template <typename T, int EPT, Access VEC>
__device__ __forceinline__ void raw_load(unsigned char* s, const T* p, int n, int lane)
{
	constexpr int BYTES = EPT * sizeof(T);
	constexpr int CH = BYTES < 16 ? BYTES : 16;
	if constexpr (VEC == kVectors && CH >= 4)
	{
#pragma unroll
		for (int i = 0; i < BYTES / CH; ++i)
		{
			const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(s + (i * 32 + lane) * CH));
			const unsigned char* src = reinterpret_cast<const unsigned char*>(p) + i * CH;
			// a source size of zero writes zeros and reads nothing
			if constexpr (CH == 16)
				asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n > 0 ? 16 : 0) : "memory");
			else
				asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(CH), "r"(n > 0 ? CH : 0) : "memory");
		}
	}
	else if constexpr (VEC == kWords && CH >= 4)
	{
#pragma unroll
		for (int e = 0; e < EPT; e += 2)
		{
			const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(s + ((e * 2 / CH) * 32 + lane) * CH + e * 2 % CH));
			asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(e < n ? p + e : p), "r"(e < n ? 4 : 0) : "memory");
		}
	}
	else
	{
		Frag<T, EPT> f;
		load_frag(f, p, n);
		constexpr int PER = CH / sizeof(T);
#pragma unroll
		for (int e = 0; e < EPT; ++e) *reinterpret_cast<T*>(s + ((e / PER) * 32 + lane) * CH + (e % PER) * sizeof(T)) = f.v[e];
	}
}
template <typename T, int EPT>
__device__ __forceinline__ void raw_read(const unsigned char* s, float* o, int lane)
{
	constexpr int BYTES = EPT * sizeof(T);
	constexpr int CH = BYTES < 16 ? BYTES : 16;
	using B = typename BitsOf<CH>::type;
	Frag<T, EPT> f;
#pragma unroll
	for (int i = 0; i < BYTES / CH; ++i) reinterpret_cast<B*>(f.v)[i] = *reinterpret_cast<const B*>(s + (i * 32 + lane) * CH);
	frag_f32(f, o);
}

// One tile (TT tokens) of B and C, which every channel of the group reads: fp32 in shared memory, [B | C][TT][NP], zero past the end of
// the sequence and past state N. Where rows allow it the elements move 16 bytes at a time, and the first PRE accesses of a thread are
// requested a tile ahead (fetch) and stored when the tile begins (store).
template <typename T, int NP, int TT, int MATRICES>
struct RowsBC
{
	static constexpr int EB = 16 / sizeof(T);
	static constexpr int TOTAL = MATRICES * TT * NP;
	static constexpr int PRE = 2;
	uint4 pre[PRE];
	const int tid, threads;  // of those that stage the tile together
	__device__ __forceinline__ RowsBC(int tid_, int threads_) : tid(tid_), threads(threads_) {}


	// pad: empty places at the head of the tile
	static __device__ __forceinline__ const T* at(const Inputs& in, const T* B, const T* C, int64_t t0, int64_t t_end, int k, int pad = 0)
	{
		const int n = k % NP, tt = (k / NP) % TT;
		const int64_t t = t0 + tt;
		if (t >= t_end || n >= in.N || tt < pad) return nullptr;
		return k < TT * NP ? B + t * in.Bs + n : C + t * in.Cs + n;
	}
	__device__ __forceinline__ void fetch(bool vec, const Inputs& in, const T* B, const T* C, int64_t t0, int64_t t_end, int pad = 0)
	{
		if (!vec) return;
#pragma unroll
		for (int i = 0; i < PRE; ++i)
		{
			const int k = (tid + i * threads) * EB;
			pre[i] = make_uint4(0, 0, 0, 0);
			if (k < TOTAL)
			{
				const T* p = at(in, B, C, t0, t_end, k, pad);
				if (p) pre[i] = *reinterpret_cast<const uint4*>(p);
			}
		}
	}
	static __device__ __forceinline__ void put(float* s, const uint4& v)
	{
		const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
		for (int j = 0; j < EB; j += 4)
			*reinterpret_cast<float4*>(s + j) = make_float4(Cvt<T>::to_f32(e[j]), Cvt<T>::to_f32(e[j + 1]), Cvt<T>::to_f32(e[j + 2]), Cvt<T>::to_f32(e[j + 3]));
	}
	__device__ __forceinline__ void store(bool vec, const Inputs& in, const T* B, const T* C, int64_t t0, int64_t t_end, float* s)
	{
		if (vec)
		{
#pragma unroll
			for (int i = 0; i < PRE; ++i)
			{
				const int k = (tid + i * threads) * EB;
				if (k < TOTAL) put(s + k, pre[i]);
			}
			for (int k = (tid + PRE * threads) * EB; k < TOTAL; k += threads * EB)
			{
				const T* p = at(in, B, C, t0, t_end, k);
				uint4 v = make_uint4(0, 0, 0, 0);
				if (p) v = *reinterpret_cast<const uint4*>(p);
				put(s + k, v);
			}
		}
		else
		{
#pragma unroll 4
			for (int k = tid; k < TOTAL; k += threads)
			{
				const T* p = at(in, B, C, t0, t_end, k);
				s[k] = p ? Cvt<T>::to_f32(*p) : 0.f;
			}
		}
	}
	// The same into ORDERS copies of the tile whose groups of four states are permuted: copy p * ORDERS / 4 holds state i ^ p of a group in
	// place i (p = 0, 2 for two orders).
	template <int ORDERS, int COPY /* elements from copy to copy */>
	__device__ __forceinline__ void store_orders(bool vec, const Inputs& in, const T* B, const T* C, int64_t t0, int64_t t_end, int pad, float* s)
	{
		auto put_orders = [&](int k, float4 v) {
#pragma unroll
			for (int o = 0; o < ORDERS; ++o)
			{
				const int p = o * 4 / ORDERS;
				const float4 a = p & 2 ? make_float4(v.z, v.w, v.x, v.y) : v;
				*reinterpret_cast<float4*>(s + o * COPY + k) = p & 1 ? make_float4(a.y, a.x, a.w, a.z) : a;
			}
		};
		if (vec)
		{
			auto put_vec = [&](int k, const uint4& raw) {
				const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
				for (int j = 0; j < EB; j += 4)
					put_orders(k + j, make_float4(Cvt<T>::to_f32(e[j]), Cvt<T>::to_f32(e[j + 1]), Cvt<T>::to_f32(e[j + 2]), Cvt<T>::to_f32(e[j + 3])));
			};
#pragma unroll
			for (int i = 0; i < PRE; ++i)
			{
				const int k = (tid + i * threads) * EB;
				if (k < TOTAL) put_vec(k, pre[i]);
			}
			for (int k = (tid + PRE * threads) * EB; k < TOTAL; k += threads * EB)
			{
				const T* p = at(in, B, C, t0, t_end, k, pad);
				uint4 v = make_uint4(0, 0, 0, 0);
				if (p) v = *reinterpret_cast<const uint4*>(p);
				put_vec(k, v);
			}
		}
		else
		{
			for (int k = tid * 4; k < TOTAL; k += threads * 4)
			{
				float v[4];
#pragma unroll
				for (int j = 0; j < 4; ++j)
				{
					const T* p = at(in, B, C, t0, t_end, k + j, pad);
					v[j] = p ? Cvt<T>::to_f32(*p) : 0.f;
				}
				put_orders(k, make_float4(v[0], v[1], v[2], v[3]));
			}
		}
	}
	// Rows that start on 16-byte boundaries and whose 16-byte pieces lie wholly before or past state N.
	static bool aligned(const b200_selective_scan_inputs* in)
	{
		return in->d_state % EB == 0 && NP % EB == 0 && aligned16(in->B) && aligned16(in->C) && in->B_stride % EB == 0 && in->C_stride % EB == 0;
	}
};

// Which channel of the warp and which four states a lane owns. Lane bit 0 is channel bit 0 and the state bits follow it: a 64- or 128-bit
// shared-memory read costs half where lanes i and i ^ 1, or i and i ^ 2, read the same address, and so the rows of B and C (shared by
// the channels) as well as the steps (shared by the lanes of a channel) do.
template <int LPC>
struct Lanes
{
	static constexpr int CW = warp_channels(LPC);
	static constexpr int SB = CW > 1 ? 2 : 1;  // lane ^ (SB << k) differs in bit k of sub; lane ^ 1 in bit 0 of cl, lane ^ (LPC << k) in bit k
	static __device__ __forceinline__ int sub(int lane) { return CW > 1 ? (lane >> 1) & (LPC - 1) : lane; }
	static __device__ __forceinline__ int cl(int lane) { return CW > 1 ? (lane & 1) | (lane / (2 * LPC) << 1) : 0; }
};

// Four per-token partial sums of a lane, summed over the LPC lanes of its channel. Two exchange steps leave each lane with fewer
// tokens instead of adding all four everywhere. On return the lane holds COUNT totals, of tokens first .. first + COUNT - 1.
template <int LPC>
struct TokenSum
{
	static constexpr int SB = Lanes<LPC>::SB;
	static constexpr int COUNT = LPC == 1 ? 4 : (LPC == 2 ? 2 : 1);
	static __device__ __forceinline__ int first(int sub) { return LPC == 1 ? 0 : (LPC == 2 ? (sub & 1) * 2 : (sub & 1) * 2 + ((sub >> 1) & 1)); }
	static __device__ __forceinline__ bool owner(int sub) { return LPC <= 4 || sub < 4; }
	static __device__ __forceinline__ void run(const float (&a)[4], int sub, float (&out)[COUNT])
	{
		if constexpr (LPC == 1)
		{
#pragma unroll
			for (int i = 0; i < 4; ++i) out[i] = a[i];
		}
		else
		{
			const bool hi = sub & 1;
			float k0 = hi ? a[2] : a[0], k1 = hi ? a[3] : a[1];
			k0 += __shfl_xor_sync(0xffffffffu, hi ? a[0] : a[2], SB);
			k1 += __shfl_xor_sync(0xffffffffu, hi ? a[1] : a[3], SB);
			if constexpr (LPC == 2)
			{
				out[0] = k0;
				out[1] = k1;
			}
			else
			{
				const bool hi2 = sub & 2;
				float k = hi2 ? k1 : k0;
				k += __shfl_xor_sync(0xffffffffu, hi2 ? k0 : k1, 2 * SB);
#pragma unroll
				for (int o = 4; o < LPC; o <<= 1) k += __shfl_xor_sync(0xffffffffu, k, o * SB);
				out[0] = k;
			}
		}
	}
};

// The four states [n0, n0 + 4) of a row of N; entries past N read zero and are not written. vec4: N and the row are multiples of 4.
__device__ __forceinline__ void load_states(bool vec4, float* h, const float* p, int n0, int N)
{
	if (vec4)
	{
		float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
		if (n0 < N) v = *reinterpret_cast<const float4*>(p + n0);
		h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
	}
	else
	{
#pragma unroll
		for (int i = 0; i < kStates; ++i) h[i] = n0 + i < N ? p[n0 + i] : 0.f;
	}
}
__device__ __forceinline__ void store_states(bool vec4, const float* h, float* p, int n0, int N)
{
	if (vec4)
	{
		if (n0 < N) *reinterpret_cast<float4*>(p + n0) = make_float4(h[0], h[1], h[2], h[3]);
	}
	else
	{
#pragma unroll
		for (int i = 0; i < kStates; ++i)
			if (n0 + i < N) p[n0 + i] = h[i];
	}
}
__device__ __forceinline__ void load_states2(bool vec4, f2* h, const float* p, int n0, int N)
{
	float v[kStates];
	load_states(vec4, v, p, n0, N);
	h[0] = pack2(v[0], v[1]);
	h[1] = pack2(v[2], v[3]);
}
__device__ __forceinline__ void store_states2(bool vec4, const f2* h, float* p, int n0, int N)
{
	const float2 a = unpack2(h[0]), b = unpack2(h[1]);
	const float v[kStates] = { a.x, a.y, b.x, b.y };
	store_states(vec4, v, p, n0, N);
}

// An element of A in units of log2: exp2(delta * a2) = exp(delta * A). An infinite one becomes the largest finite number: the empty
// places of a tile have a step of zero, and zero times infinity is not zero.
__device__ __forceinline__ float decay_unit(float a, int a_is_log)
{
	const float v = (a_is_log ? -expf(a) : a) * kLog2e;
	return v < -3.4028235e38f ? -3.4028235e38f : (v > 3.4028235e38f ? 3.4028235e38f : v);
}
// A row of A
__device__ __forceinline__ void load_decay(float* a2, const float* A, int a_is_log, int n0, int N)
{
#pragma unroll
	for (int i = 0; i < kStates; ++i)
	{
		const float a = n0 + i < N ? A[n0 + i] : 0.f;
		a2[i] = n0 + i < N ? decay_unit(a, a_is_log) : 0.f;
	}
}

// Shared memory of a CTA of the backward kernel in f16 (BackwardSmem), as a function of run-time values.
int backward_smem_bytes(int lpc, int warps);

// How the channels and tokens of a call are dealt to CTAs (a function of the sizes alone).
struct Split
{
	int warps;       // per CTA
	int nbg;         // CTAs across the channels of a group
	int nseg, seg_tokens;
};
Split split_work(int64_t batch, int64_t seqlen, int64_t dim, int64_t ngroups, int64_t d_state, bool backward);

}  // namespace sscan

int selective_scan_check(int dtype, const b200_selective_scan_inputs* in);
sscan::Inputs selective_scan_params(const b200_selective_scan_inputs* in, int nbg);

}  // namespace b200
