// What the attention kernels share on the device: the elements of the exact integer softmax, and the
// integer matrix instructions.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "sslm_types.cuh"

namespace sslm {

// One softmax element for constants that passed the gates of k_qkv_post (1 <= q_ln2 <= q_b
// < 2^24, q_c >= 0, peak = q_b^2 + q_c within the width gate): the value iexp_element()
// computes, on 32-bit words and without a branch. dq = max - score (0 <= dq < 2^32).
// z = floor(x / q_ln2) comes from one fused multiply-add that rounds toward zero onto an integer grid, with a
// reciprocal a little too small, so that it is z or z - 1 and the exact remainder tells which.
//
// The reference also refuses an element whose value leaves [0, peak] (SoftmaxRowQ15's per-element
// bound, src/intmath.cpp:870-888). Under the gates above that cannot happen, so the kernels carry
// no such test: 0 <= rem < q_ln2 <= q_b gives 1 <= base = q_b - rem <= q_b, hence
// 0 <= (base^2 + q_c) >> z <= q_b^2 + q_c = peak (and peak >= 1 because q_b >= 1).
struct IExpFast {
	uint32_t ln2, clip;     // q_ln2, 30 * q_ln2
	int32_t qb;
	int64_t qc;
	float inv_ln2;          // (1 - 2^-21) / q_ln2
};
__device__ __forceinline__ IExpFast iexp_fast_prepare(const SoftmaxConsts& k) {
	IExpFast f;
	f.ln2 = (uint32_t)k.c.q_ln2;
	f.clip = 30u * f.ln2;
	f.qb = (int32_t)k.c.q_b;
	f.qc = k.c.q_c;
	f.inv_ln2 = (1.0f / (float)f.ln2) * 0.9999995f;
	return f;
}
// The element by itself: k_attention_tile, which keeps nothing between its walks. (x = z * q_ln2 + rem, rem < q_ln2 < 2^24, z <= 30)
__device__ __forceinline__ int64_t iexp_fast(uint32_t dq, const IExpFast& f) {
	const uint32_t x = min(dq, f.clip);
	uint32_t z = (uint32_t)__float_as_int(__fmaf_rz(__uint2float_rn(x), f.inv_ln2, 8388608.0f)) - 0x4B000000u;
	uint32_t rem = x - z * f.ln2;
	if (rem >= f.ln2) {
		rem -= f.ln2;
		++z;
	}
	const int32_t base = f.qb - (int32_t)rem;
	return (int64_t)((uint64_t)((int64_t)base * (int64_t)base + f.qc) >> z);
}
// Q15 probability floor((e << 15) / tot), 0 <= e <= tot, 1 <= tot < 2^63.
//
// The row's constants scale e to 31 bits; the float product is then within pf 2^-21 + 2^-15 of the
// quotient, and its floor (one add that rounds toward zero) is the answer unless the fraction is that
// close to an integer -- at most one element in some ten thousand, and never below the first integer,
// where nearly all elements of a long row lie. Those take prob_q15.
struct ProbRow {
	unsigned long long tot;
	float c;      // 2^(15 + sh) / tot
	int sh;
};
__device__ __forceinline__ ProbRow prob_row(unsigned long long total) {
	ProbRow r;
	r.tot = total > 1ull ? total : 1ull;
	r.sh = max(0, 33 - __clzll((long long)r.tot));
	r.c = (32768.0f / (float)r.tot) * __int_as_float((127 + r.sh) << 23);
	return r;
}
// the exact form: a float quotient off by at most one, settled by one signed remainder
__device__ __forceinline__ uint32_t prob_q15(int64_t e, unsigned long long tot, float rinv) {
	const unsigned long long num = (unsigned long long)e << 15;
	uint32_t p = min(__float2uint_rz(__ll2float_rn(e) * rinv), 32768u);
	const long long r = (long long)(num - (unsigned long long)p * tot);
	p -= r < 0 ? 1u : 0u;
	p += r >= (long long)tot ? 1u : 0u;
	return p;
}
// bits 0..15 of the result: the probability, unless *unsure came out true
__device__ __forceinline__ uint32_t prob_fast(int64_t e, const ProbRow& r, bool* unsure) {
	const float pf = __uint2float_rn((uint32_t)((uint64_t)e >> r.sh)) * r.c;
	const float t = __fadd_rz(pf, 8388608.0f);
	const float off = fabsf((pf - (t - 8388608.0f)) - 0.5f), eps = fmaf(pf, 4.76837158203125e-07f, 3.2e-05f);
	*unsure = *unsure || (off > 0.5f - eps && pf > eps);
	return (uint32_t)__float_as_int(t);
}
static __device__ __noinline__ uint2 prob_pair_exact(int64_t e0, int64_t e1, unsigned long long tot) {
	const float rinv = 32768.0f / (float)tot;
	return make_uint2(prob_q15(e0, tot, rinv), prob_q15(e1, tot, rinv));
}
// A row's constants of the probability pass. pf = (base^2 + q_c) 2^-z 32768 / total in float is within
// pf 2^-21 (five roundings) + 32768 / total (the element's own floor) of the quotient, so its floor is the
// probability unless the nearest integer from 1 up is that close; those take prob_q15. Below 1 it is 0.
struct ChunkProb {
	float c, qc, eps;
};
__device__ __forceinline__ ChunkProb chunk_prob(unsigned long long total, const IExpFast& f) {
	ChunkProb p;
	p.c = 32768.0f / (float)(total > 1ull ? total : 1ull);
	p.qc = (float)f.qc;
	p.eps = p.c * 1.01f;
	return p;
}
constexpr uint32_t kBaseOfZero = 63u << 24;      // (shift, base) of an element that counts for nothing
// The element of the kernels that keep their scores; *parts, its (shift, base) word, takes the score's place and the
// probability pass reads it instead of dividing again.
__device__ __forceinline__ int64_t chunk_exp(uint32_t dq, const IExpFast& f, uint32_t* parts) {
	const uint32_t x = min(dq, f.clip);
	uint32_t z = (uint32_t)__float_as_int(__fmaf_rz(__uint2float_rn(x), f.inv_ln2, 8388608.0f)) - 0x4B000000u;
	uint32_t rem = x - z * f.ln2;
	if (rem >= f.ln2) {
		rem -= f.ln2;
		++z;
	}
	const uint32_t base = (uint32_t)f.qb - rem;      // 1 .. q_b < 2^24
	*parts = (z << 24) + base;
	return (int64_t)(((uint64_t)base * base + (uint64_t)f.qc) >> z);
}
__device__ __forceinline__ uint32_t chunk_prob_of(uint32_t parts, const ChunkProb& p, float* near) {
	const float bf = __uint2float_rn(parts & 0xFFFFFFu);
	const float pf = fmaf(bf, bf, p.qc) * __int_as_float(__float_as_int(p.c) - (int)((parts >> 24) << 23));
	const float whole = fmaxf((pf + 8388608.0f) - 8388608.0f, 1.0f);
	*near = fminf(*near, fmaf(pf, -4.76837158203125e-07f, fabsf(pf - whole)));
	return (uint32_t)__float_as_int(__fadd_rz(pf, 8388608.0f));      // (low 16 bits)
}
static __device__ __noinline__ uint4 chunk_prob_exact(uint32_t p0, uint32_t p1, uint32_t p2, uint32_t p3, int64_t qc, unsigned long long total) {
	const unsigned long long tot = total > 1ull ? total : 1ull;
	const float rinv = 32768.0f / (float)tot;
	auto one = [&](uint32_t p) {
		const uint64_t base = p & 0xFFFFFFu;
		return (p >> 24) == 63u ? 0u : prob_q15((int64_t)((base * base + (uint64_t)qc) >> (p >> 24)), tot, rinv);
	};
	return make_uint4(one(p0), one(p1), one(p2), one(p3));
}

// bytes 0 (low plane) or 1 (high plane) of four probabilities, packed into one word
__device__ __forceinline__ uint32_t pack_plane(uint32_t p0, uint32_t p1, uint32_t p2, uint32_t p3, int byte) {
	const uint32_t sel = byte ? 0x0051u : 0x0040u;
	return __byte_perm(__byte_perm(p0, p1, sel), __byte_perm(p2, p3, sel), 0x5410u);
}

// D += A(16x32, row) * B(32x8, col), int8 or (probability planes) u8 times int8
__device__ __forceinline__ void mma_s8s8_full(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
	asm volatile(
	    "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
	    : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
	    : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8_full(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
	asm volatile(
	    "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
	    : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
	    : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

}  // namespace sslm
