// The q/k/v site on a caller's tensors: int32 projections of q, k and v become rotated int8 codes of q, softmax constants, and K and V in
// the pages of the cache.
//
//   q: the row's funnel (one scale a row), or each head normed;  K: landed on its head's scale, or normed;  V: landed
//   norm of a head:  y = x 2^s with 2^23 <= max |y| <= 2^24,  root = floor(sqrt(64 sum y^2 / n)),  u = round(y floor(2^54 / root) / 2^36),
//   code = round(u gain / 2^shift). The sum is below 2^55 and the root at least 2^22.5, so its reciprocal fits 32 bits and every product 64.
//   (The shift s makes the result the same for every scale of x to one part in 2^22; a norm has no other use for the scale.)
//   rotation: pairs of channels, neighbours or rotary / 2 apart, on codes, with angles of 30 bits
//
// A thread takes four neighbouring elements (a quad), so a head is 8, 16 or 32 neighbouring lanes: what a head needs of itself (its maximum,
// its sum of squares, the other half of its pairs) is exchanged in the warp. Only the funnel's maximum needs the block. Two forms: a block a
// row, and for many rows eight rows a block.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/sslm_b200.h"
#include "sslm_kernels.h"
#include "sslm_quad.cuh"

namespace sslm {
namespace {

constexpr int kSiteMostElements = 32768;

struct SiteArgs {
	sslm_b200_qkv_site c;
	int nq, nk, total;      // quads of q, of K (and as many of V), of the row
	int lanes;              // of a head
	int q_warps, k_warps;   // of q, of K (and as many of V) when a warp has 32 quads of one of them
};

// what a row says of itself; code 0 and a position: it is worked on. (Everything but the page is asked for at once.)
struct SiteRow {
	int pos, place, page, code;
	int in_m, in_e;
};
__device__ __forceinline__ SiteRow site_row(const sslm_b200_qkv_site& a, int64_t r, bool lands) {
	const bool scaled = a.q_gain == nullptr || lands;
	SiteRow w{a.positions[r], 0, 0, 0, 1 << 30, 0};
	const int64_t m = scaled ? a.in_scales[2 * r] : (int64_t)1 << 30, e = scaled ? a.in_scales[2 * r + 1] : 0;
	const int place = lands && a.places != nullptr ? a.places[r] : w.pos, table = lands && a.table_of != nullptr ? a.table_of[r] : (int)r;
	if (w.pos == -1) return w;
	if (w.pos < 0 || w.pos >= a.num_positions) w.code = SSLM_B200_ROW_LENGTH;
	if (m < ((int64_t)1 << 30) || m >= ((int64_t)1 << 31) || e < -4096 || e > 4096) w.code = w.code != 0 ? w.code : SSLM_B200_ROW_CONSTANTS;
	else {
		w.in_m = (int)m;
		w.in_e = (int)e;
	}
	if (lands) {
		w.place = place;
		if (place < 0 || place >= a.table_pages * kPageTokens) w.code = w.code != 0 ? w.code : SSLM_B200_ROW_LENGTH;
		else if (table < 0 || table >= a.num_tables) w.code = w.code != 0 ? w.code : SSLM_B200_ROW_INDEX;
		else {
			w.page = a.pages[table * a.pages_stride + place / kPageTokens];
			if (w.page < 0 || w.page >= a.num_pages) w.code = w.code != 0 ? w.code : SSLM_B200_ROW_INDEX;
		}
	}
	return w;
}

// four elements landed on their head's scale: codes in the low word, how many were held in the high one
static __device__ __noinline__ uint64_t land_quad_exact(int32_t x0, int32_t x1, int32_t x2, int32_t x3, int64_t m, int64_t r_t, int64_t e, int64_t e_t) {
	const int32_t x[4] = {x0, x1, x2, x3};
	int c[4];
	uint32_t held = 0;
	for (int j = 0; j < 4; ++j) {
		bool over;
		const int64_t v = landing_rescale(x[j], m, r_t, e, e_t, &over, nullptr);
		c[j] = over ? (x[j] < 0 ? -127 : 127) : (int)v;
		held += over ? 1u : 0u;
	}
	return (uint64_t)held << 32 | pack4(c[0], c[1], c[2], c[3]);
}
__device__ __forceinline__ uint32_t land_quad(const int32_t (&x)[4], Scale in, int64_t e_t, int64_t r_t, uint32_t& held) {
	const Lander l = make_lander(in.m, r_t, in.e, e_t);
	if (!l.fast) {
		const uint64_t v = land_quad_exact(x[0], x[1], x[2], x[3], in.m, r_t, in.e, e_t);
		held += (uint32_t)(v >> 32);
		return (uint32_t)v;
	}
	int c[4];
#pragma unroll
	for (int j = 0; j < 4; ++j) {
		const uint64_t m = land_magnitude(abs_u32(x[j]), l);
		held += m > 127 ? 1u : 0u;
		c[j] = (int)min(m, (uint64_t)127);
		if (x[j] < 0) c[j] = -c[j];
	}
	return pack4(c[0], c[1], c[2], c[3]);
}

// the codes c at elements e to e + 3 of a head turned by a row of the tables (all lanes of the warp take part)
__device__ __forceinline__ uint32_t turn_quad(const sslm_b200_qkv_site& a, uint32_t c, int e, const int32_t* cos, const int32_t* sin, bool turned) {
	const int lane = threadIdx.x & 31, half_lanes = a.rotary >> 3;
	const uint32_t other = a.halves ? __shfl_sync(0xffffffffu, c, e < a.rotary ? (e < a.rotary / 2 ? lane + half_lanes : lane - half_lanes) : lane) : 0u;
	if (!turned || e >= a.rotary) return c;
	if (!a.halves) return rope_quad(c, *(const int2*)(cos + (e >> 1)), *(const int2*)(sin + (e >> 1)));
	const bool low = e < a.rotary / 2;
	const int at = low ? e : e - a.rotary / 2;
	const int4 cs = *(const int4*)(cos + at), sn = *(const int4*)(sin + at);
	const int co[4] = {cs.x, cs.y, cs.z, cs.w}, si[4] = {sn.x, sn.y, sn.z, sn.w};
	int out[4];
#pragma unroll
	for (int j = 0; j < 4; ++j) {
		const int mine = byte_of(c, j), theirs = byte_of(other, j);
		out[j] = rope_round(low ? (int64_t)mine * co[j] - (int64_t)theirs * si[j] : (int64_t)theirs * si[j] + (int64_t)mine * co[j]);
	}
	return pack4(out[0], out[1], out[2], out[3]);
}

// softmax constants of row r for the kv heads first, first + step, ...; true where one cannot be
static __device__ __noinline__ bool site_consts(const int64_t* khead, int64_t* consts, int kv_heads, int64_t r, Scale q, int first, int step) {
	bool bad = false;
	for (int h = first; h < kv_heads; h += step) {
		SoftmaxConsts sc;
		const bool none = softmax_consts(q, Scale{khead[2 * h], khead[2 * h + 1]}, 1, &sc) != kOk;
		int64_t* to = consts + (r * kv_heads + h) * 3;
		to[0] = none ? 0 : sc.c.q_ln2;
		to[1] = none ? 0 : sc.c.q_b;
		to[2] = none ? 0 : sc.c.q_c;
		bad = bad || none;
	}
	return bad;
}

// u = y R / 2^36 in Q15 and the code of it: R = floor(2^54 / root) below 2^32, y at most 2^24, u below 2^19
__device__ __forceinline__ uint32_t norm_reciprocal(uint64_t mean) {
	const int64_t root = max((int64_t)1, isqrt64((int64_t)mean));
	uint64_t q = (uint64_t)((double)(1ull << 54) * rcp_estimate((double)root));
	int64_t rest = (int64_t)((1ull << 54) - q * (uint64_t)root);
	while (rest < 0) { --q; rest += root; }
	while (rest >= root) { ++q; rest -= root; }
	return (uint32_t)min(q, (uint64_t)0xFFFFFFFFu);
}

// Four elements of a head as codes before they are held; a head is `lanes` lanes, and all lanes of the warp take part.
__device__ __forceinline__ void norm_quad(const int32_t (&x)[4], const int16_t* gain, int shift, int lanes, int (&code)[4], uint32_t& held) {
	uint32_t a[4], top = 0;
#pragma unroll
	for (int j = 0; j < 4; ++j) {
		a[j] = abs_u32(x[j]);
		top = max(top, a[j]);
	}
	for (int o = lanes >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
	const int up = __clz((int)max(top, 1u)) - 8;      // 23 - floor(log2 top)
	unsigned long long sum = 0;
#pragma unroll
	for (int j = 0; j < 4; ++j) {
		a[j] = up >= 0 ? a[j] << up : (a[j] + (1u << (-up - 1))) >> -up;
		sum += (unsigned long long)a[j] * a[j];
	}
	for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
	const int log_n = 33 - __clz(lanes);              // of 4 * lanes
	const uint32_t recip = norm_reciprocal(log_n <= 6 ? sum << (6 - log_n) : sum >> (log_n - 6));
	const unsigned long long half = 1ull << (shift - 1);
	const short4 g = *(const short4*)gain;
	const int gs[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
	for (int j = 0; j < 4; ++j) {
		const uint32_t u = (uint32_t)(((unsigned long long)a[j] * recip + (1ull << 35)) >> 36);
		const unsigned long long m = ((unsigned long long)u * (uint32_t)abs(gs[j]) + half) >> shift;
		const int c = (int)min(m, 128ull);
		held += c > 127 ? 1u : 0u;
		code[j] = ((x[j] < 0) != (gs[j] < 0)) ? -min(c, 127) : min(c, 127);
	}
}

// A block a row, NV quads a thread. One quad where there is a block for every SM at most, the shortest way through a row (148 rows of 16 + 2 + 2
// heads of 128 4.9 us, two quads 5.3; normed 5.5 and 6.6); two beyond, because a block does a row's scalars in every warp (300 rows 7.1, one quad
// 11.0; normed 8.9, 12.7); more only for rows that need more threads than a block has. One row: 4.6 us with 12 + 2 + 2 heads, of which the host's
// part of the call is most.
template <int NV>
__global__ void __launch_bounds__(NV == 1 ? 1024 : 512)
k_qkv_site(const __grid_constant__ SiteArgs g) {
	__shared__ uint32_t s_bank[64];
	Bank bank{s_bank, 0};
	const sslm_b200_qkv_site& a = g.c;
	const int t = threadIdx.x, T = blockDim.x, lane = t & 31, hd = a.head_dim;
	const int64_t r = blockIdx.x;
	pdl_wait();
	pdl_release();
	int32_t x[NV][4];
#pragma unroll
	for (int v = 0; v < NV; ++v) {
		const int i = t + v * T;
		x[v][0] = x[v][1] = x[v][2] = x[v][3] = 0;
		if (i < g.nq) load_quad(a.q + r * a.q_stride + 4 * i, x[v]);
		else if (i < g.nq + g.nk) load_quad(a.k + r * a.k_stride + 4 * (i - g.nq), x[v]);
		else if (i < g.total) load_quad(a.v + r * a.v_stride + 4 * (i - g.nq - g.nk), x[v]);
	}
	const SiteRow w = site_row(a, r, g.nk > 0);      // (all threads alike)
	if (w.pos == -1 || w.code != 0) {
		if (t == 0 && a.row_status != nullptr) a.row_status[r] = w.code;
		return;
	}
	const Scale site{a.q_site_m, a.q_site_e};
	QuadFunnel fp{};
	fp.out = site;
	if (g.nq > 0 && a.q_gain == nullptr) {
		uint32_t top = 0;
#pragma unroll
		for (int v = 0; v < NV; ++v)
			if (t + v * T < g.nq) top = max(max(max(top, abs_u32(x[v][0])), abs_u32(x[v][1])), max(abs_u32(x[v][2]), abs_u32(x[v][3])));
		const Scale scale{w.in_m, w.in_e};
		const FunnelFold fold = funnel_prefold(&scale, 1, site);
		fp = quad_funnel(T > 32 ? block_max_u32(top, bank) : __reduce_max_sync(0xffffffffu, top), fold);      // (canonical scales: never refused)
	}
	const int slot = w.place % kPageTokens;
	const int64_t turn = (int64_t)w.pos * (a.rotary >> 1);
	const Scale in{w.in_m, w.in_e};
	uint32_t held = 0;
#pragma unroll
	for (int v = 0; v < NV; ++v) {
		const int i = t + v * T, e = (4 * i) & (hd - 1);
		const bool is_q = i < g.nq, is_k = !is_q && i < g.nq + g.nk, is_v = !is_q && !is_k && i < g.total;
		const int head = is_q ? 0 : ((i - g.nq - (is_k ? 0 : g.nk)) * 4) / hd;      // of K or V
		uint32_t c = 0;
		const bool normed = (is_q && a.q_gain != nullptr) || (is_k && a.k_gain != nullptr);
		if (a.q_gain != nullptr || a.k_gain != nullptr) {
			int lc[4];
			uint32_t over = 0;
			const int16_t* gain = normed ? (is_q ? a.q_gain : a.k_gain) : (a.q_gain != nullptr ? a.q_gain : a.k_gain);
			norm_quad(x[v], gain + e, normed ? (is_q ? a.q_shift : a.k_shift) : 1, g.lanes, lc, over);
			if (normed) {
				c = pack4(lc[0], lc[1], lc[2], lc[3]);
				if (is_k) held += over;
			}
		}
		if (is_q && !normed) c = code_quad(x[v], fp);
		if (!is_q && !normed && i < g.total) {
			const int64_t* rec = (is_k ? a.k_landing : a.v_landing) + 3 * head;
			const int64_t e_t = rec[1], r_t = rec[2];
			c = land_quad(x[v], in, e_t, r_t, held);
		}
		c = turn_quad(a, c, e, a.cos + turn, a.sin + turn, is_q || is_k);
		if (is_q) {
			*(uint32_t*)(a.q_codes + r * a.q_codes_stride + 4 * i) = c;
		} else if (is_k) {
			*(uint32_t*)(a.kv + ((2 * (int64_t)head * a.num_pages + (int64_t)w.page) * kPageTokens + slot) * hd + e) = c;
		} else if (is_v) {
			int8_t* to = a.kv + (((2 * (int64_t)head + 1) * a.num_pages + (int64_t)w.page) * hd + e) * kPageTokens + slot;
#pragma unroll
			for (int j = 0; j < 4; ++j) to[j * kPageTokens] = (int8_t)byte_of(c, j);
		}
	}
	if (g.nk > 0 && a.saturations != nullptr) {
		held = T > 32 ? block_sum_u32(held, bank) : __reduce_add_sync(0xffffffffu, held);
		if (t == 0) a.saturations[r] = (int32_t)held;
	}
	// the last warp's lanes: scales, softmax constants, status
	if (t < T - 32) return;
	bool bad = false;
	if (g.nq > 0) {
		if (lane == 0 && a.q_scales != nullptr) {
			a.q_scales[2 * r] = fp.out.m;
			a.q_scales[2 * r + 1] = fp.out.e;
		}
		if (a.consts != nullptr) bad = site_consts(a.khead, a.consts, a.kv_heads, r, fp.out, lane, 32);
	}
	bad = __any_sync(0xffffffffu, bad);
	if (lane == 0 && a.row_status != nullptr) a.row_status[r] = bad ? SSLM_B200_ROW_SOFTMAX : 0;
}

// Landing and rotation of many rows find their integers in float, and leave to the integer forms what is too close to a tie to know.
//   landing:  v = x rho, rho = m r_t / 2^k. Five roundings (of x, m, r_t, and two products) move a v of at most 128 by 128 * 2^-24 each, 3.9e-5 in all.
//   rotation: v = a c - b s, c and s in Q30 rounded to 24 bits (|c| <= 2: by 2^-24), |a|, |b| <= 127. Both terms together move by
//             2 * 127 * 2^-24, b s rounds by 2^-17 and a result that is not held by 2^-18: 2.7e-5.
// The distance to the nearest integer is exact (both are multiples of the float's last bit, and it is at most a half).
constexpr float kLandTie = 0.49995f, kTurnTie = 0.49997f;
// rf, ef: r_t and e_t, rf zero where they are out of range; mf: m
__device__ __forceinline__ float land_factor(float mf, int e, float rf, int ef) {
	const int k = 62 - (e - ef);
	return k >= 33 && k <= 94 ? mf * rf * __int_as_float((127 - k) << 23) : 0.0f;
}
// four elements as whole floats from -127 to 127; returns how near to a tie the nearest is (1 where this form does not apply)
__device__ __forceinline__ float land_floats(const int4& x, float rho, float (&code)[4], uint32_t& held) {
	const int xs[4] = {x.x, x.y, x.z, x.w};
	float far = rho > 0.0f ? 0.0f : 1.0f;
#pragma unroll
	for (int j = 0; j < 4; ++j) {
		const float v = fminf(fmaxf(__int2float_rn(xs[j]) * rho, -200.0f), 200.0f), q = (v + kRoundMagic) - kRoundMagic;
		far = fmaxf(far, fabsf(v - q));
		held += fabsf(q) > 127.0f ? 1u : 0u;
		code[j] = fminf(fmaxf(q, -127.0f), 127.0f);
	}
	return far;
}
__device__ __forceinline__ uint32_t pack_floats(const float (&code)[4]) {
	return pack4(__float_as_int(code[0] + kRoundMagic), __float_as_int(code[1] + kRoundMagic), __float_as_int(code[2] + kRoundMagic), __float_as_int(code[3] + kRoundMagic));
}
// the integer form
static __device__ __noinline__ uint32_t turn_quad_exact(uint32_t c, uint32_t other, const int32_t* cos, const int32_t* sin, bool halves, bool low) {
	if (!halves) return rope_quad(c, make_int2(cos[0], cos[1]), make_int2(sin[0], sin[1]));
	int out[4];
	for (int j = 0; j < 4; ++j) {
		const int64_t mine = byte_of(c, j), theirs = byte_of(other, j);
		out[j] = rope_round(low ? mine * cos[j] - theirs * sin[j] : theirs * sin[j] + mine * cos[j]);
	}
	return pack4(out[0], out[1], out[2], out[3]);
}
// what a lane's quads have in common
struct TurnLane {
	int half, angle, partner;      // words of a table row, the quad's first, the lane with the other half
	bool turned, low;
};
__device__ __forceinline__ TurnLane turn_lane(const sslm_b200_qkv_site& a, int e) {
	const int lane = threadIdx.x & 31, half = a.rotary >> 1, half_lanes = a.rotary >> 3;
	const bool low = e < half, turned = e < a.rotary;
	return TurnLane{half, a.halves ? (low ? e : e - half) : e >> 1, turned && a.halves ? (low ? lane + half_lanes : lane - half_lanes) : lane, turned, low};
}
// U rows' quads turned: the tables' rows, cosines then sines, step apart
template <int U>
__device__ __forceinline__ void turn_floats(const sslm_b200_qkv_site& a, const float (&code)[U][4], const TurnLane& l, const int32_t* turn, int step, uint32_t (&c)[U]) {
	float other[U][4] = {}, far = 0.0f;
	if (a.halves) {
#pragma unroll
		for (int u = 0; u < U; ++u)
#pragma unroll
			for (int j = 0; j < 4; ++j) other[u][j] = __shfl_sync(0xffffffffu, code[u][j], l.partner);
	}
	if (!l.turned) {
#pragma unroll
		for (int u = 0; u < U; ++u) c[u] = pack_floats(code[u]);
		return;
	}
	turn += l.angle;
#pragma unroll
	for (int u = 0; u < U; ++u) {
		float v[4];      // 30 bits behind the point
		if (a.halves) {
			const int4 co = *(const int4*)(turn + u * step), si = *(const int4*)(turn + u * step + l.half);
			const int cs[4] = {co.x, co.y, co.z, co.w}, sn[4] = {si.x, si.y, si.z, si.w};
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				const float b = other[u][j] * __int2float_rn(sn[j]);
				v[j] = fmaf(code[u][j], __int2float_rn(cs[j]), l.low ? -b : b);
			}
		} else {
			const int2 co = *(const int2*)(turn + u * step), si = *(const int2*)(turn + u * step + l.half);
			const float c0 = __int2float_rn(co.x), c1 = __int2float_rn(co.y), s0 = __int2float_rn(si.x), s1 = __int2float_rn(si.y);
			v[0] = fmaf(code[u][0], c0, -(code[u][1] * s0));
			v[1] = fmaf(code[u][0], s0, code[u][1] * c0);
			v[2] = fmaf(code[u][2], c1, -(code[u][3] * s1));
			v[3] = fmaf(code[u][2], s1, code[u][3] * c1);
		}
		int out[4];
		constexpr float top = 127.0f * (1 << 30), q30 = 1.0f / (1 << 30);
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			v[j] = fminf(fmaxf(v[j], -top), top);
			const float m = fmaf(v[j], q30, kRoundMagic);
			far = fmaxf(far, fabsf(fmaf(v[j], q30, kRoundMagic - m)));
			out[j] = __float_as_int(m);
		}
		c[u] = pack4(out[0], out[1], out[2], out[3]);
	}
	if (far > kTurnTie)
#pragma unroll
		for (int u = 0; u < U; ++u) c[u] = turn_quad_exact(pack_floats(code[u]), pack_floats(other[u]), turn + u * step, turn + u * step + l.half, a.halves != 0, l.low);
}

// kRows rows a block. A warp has 32 quads (whole heads) of q, of K or of V in all of them; the last warp has what the rows say of
// themselves, the funnel's scalars and the softmax constants, a lane a row. It takes less than a block a row with two quads a thread where those
// blocks no longer fit the device at once, from about 2,048 quads for every SM on and four rows (5,000 where q is normed, whose roots the warps do one behind the
// other). Eleven widths, 1,536 to 12,288 quads an SM, this form / a block a row, us:
//   12 + 2 + 2 heads of 128   593 rows 9.0 / 8.4   723 9.2 / 9.6   917 8.7 / 10.6   1,777 13.0 / 17.3   3,553 23.0 / 31.0
//    4 + 2 + 2 heads of 32  2,368 rows 6.8 / 6.0   4,737 7.9 / 9.3   9,473 12.3 / 15.4   28,417 29.7 / 40.9
//   20 + 4 + 4 heads of 128   413 rows 11.6 / 10.9   677 12.3 / 15.0   2,030 22.7 / 34.7
//   q and K normed: 12 + 2 + 2 of 128 1,185 rows 22.7 / 17.5, 1,777 23.1 / 23.8, 3,553 41.2 / 43.4; 4 + 2 + 2 of 32 4,737 rows 13.7 / 12.4, 14,209 31.4 / 29.8, 28,417
//   52.2 / 57.3; 16 + 2 + 2 of 128 1,157 rows 16.6 / 19.5. K alone: 12 + 2 + 2 of 128 723 rows 13.4 / 13.6, 1,185 17.5 / 19.8.
// Both go up by steps, as their blocks fill the device once more, so near the border either may be a tenth ahead.
// The floor of 8,191 rows is 13.6 us of memory traffic; what bounds it are instructions, about 140 for 32 quads and a row, half of them on the half-rate
// pipe of comparisons and conversions (9,000 of a block's 14,000 cycles, with two blocks an SM), and the chain in front of them (positions and tables,
// maxima, scalars: 4,400). Two blocks of 17 warps leave 56 registers, so 92 bytes are stored and 192 loaded again. Measured and left: 4 rows a block (56 us), 16
// (one block an SM: 102), three blocks an SM with 32 registers (55), one or four rows side by side (46.6, 65 where two took 45), the rotation in integers
// (58 where it took 53).
constexpr int kRows = 8, kMostColumns = 31;
struct SiteShared {
	uint32_t top[32 * kRows], held[kRows], live;
	int page[kRows], slot[kRows], in_m[kRows], in_e[kRows];      // (page: -1 where the row is not worked on)
	float4 funnel[kRows];      // f, f_lo and d (as bits)
};
template <bool NORMS, int MOST, int MIN>
__global__ void __launch_bounds__(MOST, MIN) k_qkv_site_rows(const __grid_constant__ SiteArgs g) {
	extern __shared__ __align__(16) int32_t s_x[];      // a thread's quads: kRows, x_step apart; then the tables' rows
	__shared__ SiteShared s;
	const sslm_b200_qkv_site& a = g.c;
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5, hd = a.head_dim, own = lane % kRows;      // (own: the lane's row)
	const int64_t r0 = (int64_t)blockIdx.x * kRows;
	const int rows = (int)min((int64_t)kRows, a.rows - r0), half = a.rotary >> 1;
	const bool is_q = warp < g.q_warps, is_k = !is_q && warp < g.q_warps + g.k_warps, last = warp == g.q_warps + 2 * g.k_warps, is_v = !is_q && !is_k && !last;
	constexpr int U = 2;      // rows side by side: their instructions fill each other's waits, and they share the tests for ties
	const bool funnel = g.nq > 0 && a.q_gain == nullptr;
	const int x_step = 128 * (g.q_warps + 2 * g.k_warps), turn_step = 2 * half;
	int32_t *x_at = s_x + 4 * t, *s_turn = s_x + kRows * x_step;
	pdl_wait();
	pdl_release();
	if (last) {
		const SiteRow w = site_row(a, r0 + min(own, rows - 1), g.nk > 0);
		const bool lives = own < rows && w.pos != -1 && w.code == 0;
		const uint32_t live = __ballot_sync(0xffffffffu, lives) & ((1u << kRows) - 1u);
		const Scale in{lives ? w.in_m : 1 << 30, lives ? w.in_e : 0}, site{a.q_site_m, a.q_site_e};
		if (lane < kRows) {
			s.held[lane] = 0;
			s.page[lane] = lives ? w.page : -1;
			s.slot[lane] = w.place % kPageTokens;
			s.in_m[lane] = (int)in.m;
			s.in_e[lane] = (int)in.e;
			if (lane == 0) s.live = live;
		}
		FunnelFold fold{};
		if (funnel) fold = funnel_prefold(&in, 1, site);
		__syncthreads();
		Scale out = site;
		if (funnel) {
			uint32_t top = 0;
			for (int k = lane; k < g.q_warps * kRows; k += 32) top = max(top, s.top[k]);
#pragma unroll
			for (int o = kRows; o < 32; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
			const QuadFunnel fp = quad_funnel(top, fold);      // (canonical scales: never refused)
			if (lane < kRows) s.funnel[lane] = make_float4(fp.f, fp.f_lo, __uint_as_float(fp.d), 0.0f);
			out = fp.out;
			asm volatile("bar.sync 1, %0;" ::"r"(32 * (g.q_warps + 1)) : "memory");
		}
		bool bad = false;
		const int64_t row = r0 + own;
		if (g.nq > 0 && lives) {
			if (lane < kRows && a.q_scales != nullptr) {
				a.q_scales[2 * row] = out.m;
				a.q_scales[2 * row + 1] = out.e;
			}
			if (a.consts != nullptr) bad = site_consts(a.khead, a.consts, a.kv_heads, row, out, lane / kRows, 32 / kRows);
		}
		uint32_t none = __ballot_sync(0xffffffffu, bad);
#pragma unroll
		for (int o = 16; o >= kRows; o >>= 1) none |= none >> o;
		if (lane < rows && a.row_status != nullptr) a.row_status[row] = w.code != 0 ? w.code : (((none >> lane) & 1) ? SSLM_B200_ROW_SOFTMAX : 0);
		return;
	}
	const int i = 32 * (is_q ? warp : (is_k ? warp - g.q_warps : warp - g.q_warps - g.k_warps)) + lane;
	const bool in = i < (is_q ? g.nq : g.nk);
	{
		const int64_t stride = is_q ? a.q_stride : (is_k ? a.k_stride : a.v_stride);
		const int32_t* from = (is_q ? a.q : (is_k ? a.k : a.v)) + r0 * stride + 4 * i;
		const uint32_t to = (uint32_t)__cvta_generic_to_shared(x_at);
		const int pos = a.positions[r0 + min(own, rows - 1)];
		if (in && rows == kRows) {
#pragma unroll
			for (int r = 0; r < kRows; ++r, from += stride) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 4 * r * x_step), "l"(from) : "memory");
		} else {
			for (int r = 0; r < kRows; ++r, from += stride) {
				if (in && r < rows) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 4 * r * x_step), "l"(from) : "memory");
				else *(int4*)(x_at + r * x_step) = make_int4(0, 0, 0, 0);
			}
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
		// the rows of the tables, 16 bytes a thread
		const int32_t* angles = (const int32_t*)a.cos + (int64_t)pos * half;
		const int64_t sines = a.sin - a.cos;
		if (pos >= 0 && pos < a.num_positions)
			for (int k = 4 * (t / kRows); k < turn_step; k += x_step / (4 * kRows) * 4)
				asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(s_turn + own * turn_step + k)), "l"(k < half ? angles + k : angles + sines + (k - half)) : "memory");
		asm volatile("cp.async.commit_group;" ::: "memory");
		asm volatile("cp.async.wait_group 1;" ::: "memory");      // (the quads: a thread reads what it copied itself)
	}
	if (funnel && is_q) {
		uint32_t mine = 0;
#pragma unroll
		for (int r = 0; r < kRows; ++r) {
			const int4 x = *(const int4*)(x_at + r * x_step);
			const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(abs_u32(x.x), abs_u32(x.y)), max(abs_u32(x.z), abs_u32(x.w))));
			mine = lane == r ? top : mine;
		}
		if (lane < kRows) s.top[warp * kRows + lane] = mine;
	}
	asm volatile("cp.async.wait_group 0;" ::: "memory");
	__syncthreads();
	const uint32_t live = s.live;
	if (funnel && is_q) asm volatile("bar.sync 1, %0;" ::"r"(32 * (g.q_warps + 1)) : "memory");
	const int e = (4 * i) & (hd - 1);
	if (is_q) {
		const TurnLane l = turn_lane(a, e);
		int8_t* to = a.q_codes + r0 * a.q_codes_stride + 4 * i;
		for (int r = 0; r < kRows; r += U) {
			int32_t x[U][4];
			float code[U][4];
#pragma unroll
			for (int u = 0; u < U; ++u) {
				const int4 xv = *(const int4*)(x_at + (r + u) * x_step);
				x[u][0] = xv.x; x[u][1] = xv.y; x[u][2] = xv.z; x[u][3] = xv.w;
			}
			if (NORMS && a.q_gain != nullptr) {
#pragma unroll
				for (int u = 0; u < U; ++u) {
					int lc[4];
					uint32_t over = 0;
					norm_quad(x[u], a.q_gain + e, a.q_shift, g.lanes, lc, over);
#pragma unroll
					for (int j = 0; j < 4; ++j) code[u][j] = __int2float_rn(lc[j]);
				}
			} else {
				QuadFunnel f[U];
				int near[U][4];
				float far = 0.0f;
#pragma unroll
				for (int u = 0; u < U; ++u) {
					const float4 row = s.funnel[r + u];
					f[u].f = row.x;
					f[u].f_lo = row.y;
					f[u].d = __float_as_uint(row.z);
					far = fmaxf(far, code_quad_try(x[u], f[u], near[u]));
				}
				if (far > kNearTie)
#pragma unroll
					for (int u = 0; u < U; ++u) code_quad_settle(x[u], f[u], near[u]);
#pragma unroll
				for (int u = 0; u < U; ++u)
#pragma unroll
					for (int j = 0; j < 4; ++j) code[u][j] = __int_as_float(near[u][j]) - kRoundMagic;
			}
			uint32_t c[U];
			turn_floats(a, code, l, s_turn + r * turn_step, turn_step, c);
#pragma unroll
			for (int u = 0; u < U; ++u, to += a.q_codes_stride)
				if (in && ((live >> (r + u)) & 1)) *(uint32_t*)to = c[u];
		}
		return;
	}
	{
		const int head = 4 * min(i, g.nk - 1) / hd;
		const int64_t* rec = (is_k ? a.k_landing : a.v_landing) + 3 * head;
		const bool normed = NORMS && is_k && a.k_gain != nullptr;
		float rf = 0.0f;      // r_t, zero where the float form does not apply
		uint32_t r_less = 0;  // r_t - 1
		int ef = 0;
		if (!normed) {
			const int64_t e_t = rec[1], r_t = rec[2];
			if (r_t > 0 && r_t <= ((int64_t)1 << 32) && e_t > -(1 << 24) && e_t < (1 << 24)) {
				rf = __ll2float_rn(r_t);
				r_less = (uint32_t)(r_t - 1);
				ef = (int)e_t;
			}
		}
		int8_t* plane = a.kv + (2 * (int64_t)head + (is_v ? 1 : 0)) * a.num_pages * (kPageTokens * hd);
		const TurnLane l = turn_lane(a, e);
		for (int r = 0; r < kRows; r += U) {
			int4 x[U];
			float code[U][4];
			uint32_t held[U], c[U];
#pragma unroll
			for (int u = 0; u < U; ++u) {
				x[u] = *(const int4*)(x_at + (r + u) * x_step);
				held[u] = 0;
			}
			if (normed) {
#pragma unroll
				for (int u = 0; u < U; ++u) {
					const int32_t xs[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
					int lc[4];
					norm_quad(xs, a.k_gain + e, a.k_shift, g.lanes, lc, held[u]);
#pragma unroll
					for (int j = 0; j < 4; ++j) code[u][j] = __int2float_rn(lc[j]);
				}
			} else {
				float far = 0.0f;
				int in_m[U], in_e[U];
#pragma unroll
				for (int u = 0; u < U; ++u) {
					in_m[u] = s.in_m[r + u];
					in_e[u] = s.in_e[r + u];
					const float at = land_floats(x[u], land_factor(__int2float_rn(in_m[u]), in_e[u], rf, ef), code[u], held[u]);
					if ((live >> (r + u)) & 1) far = fmaxf(far, at);
				}
				if (far > kLandTie)
#pragma unroll
					for (int u = 0; u < U; ++u) {
						const uint64_t v = land_quad_exact(x[u].x, x[u].y, x[u].z, x[u].w, in_m[u], rf > 0.0f ? (int64_t)r_less + 1 : rec[2], in_e[u], rf > 0.0f ? (int64_t)ef : rec[1]);
						held[u] = (uint32_t)(v >> 32);
#pragma unroll
						for (int j = 0; j < 4; ++j) code[u][j] = (float)byte_of((uint32_t)v, j);
					}
			}
			if (is_k) {
				turn_floats(a, code, l, s_turn + r * turn_step, turn_step, c);
#pragma unroll
				for (int u = 0; u < U; ++u) {
					const int64_t token = (int64_t)s.page[r + u] * kPageTokens + s.slot[r + u];
					if (in && ((live >> (r + u)) & 1)) *(uint32_t*)(plane + token * hd + e) = c[u];
				}
			} else {
#pragma unroll
				for (int u = 0; u < U; ++u) x_at[(r + u) * x_step] = (int32_t)pack_floats(code[u]);
			}
			uint32_t any = 0;
#pragma unroll
			for (int u = 0; u < U; ++u) any |= held[u];
			if (a.saturations != nullptr && __any_sync(0xffffffffu, in && any != 0))
#pragma unroll
				for (int u = 0; u < U; ++u) {
					held[u] = __reduce_add_sync(0xffffffffu, in ? held[u] : 0u);
					if (lane == 0) atomicAdd(&s.held[r + u], held[u]);
				}
		}
		// V has the tokens of a page side by side: four rows on neighbouring places are one word
		if (is_v) {
			const int page = s.page[own], slot = s.slot[own], next = min(own + 1, kRows - 1);
			const uint32_t goes_on = __ballot_sync(0xffffffffu, page >= 0 && own + 1 < kRows && s.page[next] == page && s.slot[next] == slot + 1);      // (row r + 1 behind row r)
			for (int r = 0; r < kRows;) {
				const int at = s.slot[r];
				int8_t* to = plane + ((int64_t)s.page[r] * hd + e) * kPageTokens + at;
				const uint32_t c0 = (uint32_t)x_at[r * x_step];
				if ((at & 3) == 0 && (goes_on >> r & 7u) == 7u) {
					const uint32_t c1 = (uint32_t)x_at[(r + 1) * x_step], c2 = (uint32_t)x_at[(r + 2) * x_step], c3 = (uint32_t)x_at[(r + 3) * x_step];
					const uint32_t a0 = __byte_perm(c0, c1, 0x5140), a1 = __byte_perm(c2, c3, 0x5140);
					const uint32_t b0 = __byte_perm(c0, c1, 0x7362), b1 = __byte_perm(c2, c3, 0x7362);
					if (in) {
						*(uint32_t*)to = __byte_perm(a0, a1, 0x5410);
						*(uint32_t*)(to + kPageTokens) = __byte_perm(a0, a1, 0x7632);
						*(uint32_t*)(to + 2 * kPageTokens) = __byte_perm(b0, b1, 0x5410);
						*(uint32_t*)(to + 3 * kPageTokens) = __byte_perm(b0, b1, 0x7632);
					}
					r += 4;
					continue;
				}
				if (in && ((live >> r) & 1))
#pragma unroll
					for (int j = 0; j < 4; ++j) to[j * kPageTokens] = (int8_t)byte_of(c0, j);
				++r;
			}
		}
	}
	if (a.saturations != nullptr) {
		asm volatile("bar.sync 2, %0;" ::"r"(64 * g.k_warps) : "memory");      // (the warps of K and V)
		if (is_k && i < kRows && ((live >> i) & 1)) a.saturations[r0 + i] = (int32_t)s.held[i];
	}
}

template <int NV>
cudaError_t site_launch(const SiteArgs& g, cudaStream_t st) {
	const int threads = ((g.total + NV - 1) / NV + 31) & ~31;
	return launch_pdl(k_qkv_site<NV>, dim3(g.c.rows), dim3(threads), 0, st, g);
}

template <bool NORMS, int MOST, int MIN>
cudaError_t site_launch_rows(const SiteArgs& g, cudaStream_t st) {
	static PerDeviceOnce once;
	const cudaError_t e = once_per_device(once, [] { return cudaFuncSetAttribute(k_qkv_site_rows<NORMS, MOST, MIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRows * (MOST * 16 + 512)); });
	if (e != cudaSuccess) return e;
	const int threads = 32 * (g.q_warps + 2 * g.k_warps + 1);
	return launch_pdl(k_qkv_site_rows<NORMS, MOST, MIN>, dim3((g.c.rows - 1) / kRows + 1), dim3(threads), kRows * ((threads - 32) * 16 + g.c.rotary * 4), st, g);
}

}  // namespace
}  // namespace sslm

using namespace sslm;

extern "C" sslm_status sslm_b200_qkv_site_resident(const sslm_b200_qkv_site* call, void* stream) {
	if (!call || call->struct_size != sizeof(sslm_b200_qkv_site)) return SSLM_INVALID_ARGUMENT;
	const sslm_b200_qkv_site& c = *call;
	const bool lands = c.k != nullptr || c.v != nullptr;
	if (c.rows < 0 || c.heads < 0 || c.kv_heads < 1 || (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) || c.reserved != 0) return SSLM_INVALID_ARGUMENT;
	if (c.heads > kSiteMostElements || c.kv_heads > kSiteMostElements || ((int64_t)c.heads + 2 * (int64_t)c.kv_heads) * c.head_dim > kSiteMostElements) return SSLM_INVALID_ARGUMENT;
	if (c.rotary < 0 || c.rotary > c.head_dim || (c.rotary & 7) != 0 || c.num_positions < 0 || (c.halves != 0 && c.halves != 1)) return SSLM_INVALID_ARGUMENT;
	if (c.q_stride < (int64_t)c.heads * c.head_dim || c.k_stride < (int64_t)c.kv_heads * c.head_dim || c.v_stride < (int64_t)c.kv_heads * c.head_dim) return SSLM_INVALID_ARGUMENT;
	if (c.q_codes_stride < (int64_t)c.heads * c.head_dim) return SSLM_INVALID_ARGUMENT;
	if ((c.q_gain && (c.q_shift < 1 || c.q_shift > 62)) || (c.k_gain && (c.k_shift < 1 || c.k_shift > 62))) return SSLM_INVALID_ARGUMENT;
	if (c.num_tables < 0 || c.table_pages < 0 || c.table_pages > (1 << 26) || c.pages_stride < c.table_pages || c.num_pages < 0 || c.num_pages > 0x7FFFFFFF) return SSLM_INVALID_ARGUMENT;
	if (c.q_site_m < ((int64_t)1 << 30) || c.q_site_m >= ((int64_t)1 << 31) || c.q_site_e < -4096 || c.q_site_e > 4096) return SSLM_INVALID_ARGUMENT;
	if (c.rows == 0) return SSLM_OK;
	const bool turns = c.heads > 0 && c.q != nullptr;
	if (!turns && !lands) return SSLM_INVALID_ARGUMENT;
	if (!c.positions || (c.rotary > 0 && (!c.cos || !c.sin)) || (c.q && !c.q_codes) || (c.consts && !c.khead)) return SSLM_INVALID_ARGUMENT;
	if (lands && (!c.k || !c.v || !c.kv || !c.pages || (!c.k_gain && !c.k_landing) || !c.v_landing)) return SSLM_INVALID_ARGUMENT;
	if ((lands || !c.q_gain) && !c.in_scales) return SSLM_INVALID_ARGUMENT;
	if (lands && !c.table_of && c.num_tables < c.rows) return SSLM_INVALID_ARGUMENT;
	for (const void* p : {(const void*)c.q, (const void*)c.k, (const void*)c.v, (const void*)c.cos, (const void*)c.sin, (const void*)c.kv})
		if ((uintptr_t)p & 15) return SSLM_MISALIGNED_BUFFER;
	if ((c.q_stride | c.k_stride | c.v_stride | c.q_codes_stride) & 3) return SSLM_MISALIGNED_BUFFER;
	for (const void* p : {(const void*)c.positions, (const void*)c.places, (const void*)c.table_of, (const void*)c.pages, (const void*)c.q_codes, (const void*)c.saturations,
	                      (const void*)c.row_status})
		if ((uintptr_t)p & 3) return SSLM_MISALIGNED_BUFFER;
	for (const void* p : {(const void*)c.in_scales, (const void*)c.q_gain, (const void*)c.k_gain, (const void*)c.k_landing, (const void*)c.v_landing, (const void*)c.khead,
	                      (const void*)c.q_scales, (const void*)c.consts})
		if ((uintptr_t)p & 7) return SSLM_MISALIGNED_BUFFER;
	SiteArgs g{};
	g.c = c;
	g.lanes = c.head_dim / 4;
	g.nq = turns ? c.heads * g.lanes : 0;
	g.nk = lands ? c.kv_heads * g.lanes : 0;
	g.total = g.nq + 2 * g.nk;
	g.q_warps = (g.nq + 31) / 32;
	g.k_warps = (g.nk + 31) / 32;
	const cudaStream_t st = (cudaStream_t)stream;
	const int columns = g.q_warps + 2 * g.k_warps;
	const bool norms = c.q_gain != nullptr || c.k_gain != nullptr;
	cudaError_t e;
	const int64_t sms = sm_count(), quads = (int64_t)c.rows * g.total;
	if (c.rows >= kRows / 2 * sms && quads > (turns && c.q_gain != nullptr ? 5000 : 2048) * sms && columns <= kMostColumns) {
		if (columns <= 16) e = norms ? site_launch_rows<true, 32 * 17, 2>(g, st) : site_launch_rows<false, 32 * 17, 2>(g, st);
		else e = norms ? site_launch_rows<true, 1024, 1>(g, st) : site_launch_rows<false, 1024, 1>(g, st);
	} else if (g.total <= 1024) e = c.rows <= sm_count() ? site_launch<1>(g, st) : site_launch<2>(g, st);
	else e = g.total <= 2048 ? site_launch<4>(g, st) : site_launch<16>(g, st);
	if (e != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}
