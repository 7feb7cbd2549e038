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
// its sum of squares, the other half of its pairs) is exchanged in the warp. Only the funnel's maximum needs the block.
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
};

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
	// the row's record (all threads alike)
	const int pos = a.positions[r];
	int code = 0, place = 0;
	int64_t page = 0;
	Scale in{(int64_t)1 << 30, 0};
	if (pos != -1) {
		if (pos < 0 || pos >= a.num_positions) code = SSLM_B200_ROW_LENGTH;
		if (a.q_gain == nullptr || g.nk > 0) {
			in = Scale{a.in_scales[2 * r], a.in_scales[2 * r + 1]};
			if (in.m < ((int64_t)1 << 30) || in.m >= ((int64_t)1 << 31) || in.e < -4096 || in.e > 4096) code = code != 0 ? code : SSLM_B200_ROW_CONSTANTS;
		}
		if (g.nk > 0) {
			place = a.places != nullptr ? a.places[r] : pos;
			const int table = a.table_of != nullptr ? a.table_of[r] : (int)r;
			if (place < 0 || place >= a.table_pages * kPageTokens) code = code != 0 ? code : SSLM_B200_ROW_LENGTH;
			else if (table < 0 || table >= a.num_tables) code = code != 0 ? code : SSLM_B200_ROW_INDEX;
			else {
				page = a.pages[table * a.pages_stride + place / kPageTokens];
				if (page < 0 || page >= a.num_pages) code = code != 0 ? code : SSLM_B200_ROW_INDEX;
			}
		}
	}
	if (pos == -1 || code != 0) {
		if (t == 0 && a.row_status != nullptr) a.row_status[r] = code;
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
		const FunnelFold fold = funnel_prefold(&in, 1, site);
		fp = quad_funnel(T > 32 ? block_max_u32(top, bank) : __reduce_max_sync(0xffffffffu, top), fold);      // (canonical scales: never refused)
	}
	const int half_lanes = a.rotary >> 3, slot = place % kPageTokens;
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
			const Lander l = make_lander(in.m, r_t, in.e, e_t);
			int lc[4];
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				bool s1;
				if (l.fast) {
					const uint64_t m = land_magnitude(abs_u32(x[v][j]), l);
					s1 = m > 127;
					lc[j] = s1 ? 127 : (int)m;
					if (x[v][j] < 0) lc[j] = -lc[j];
				} else {
					const int64_t m = landing_rescale(x[v][j], in.m, r_t, in.e, e_t, &s1, nullptr);
					lc[j] = s1 ? (x[v][j] < 0 ? -127 : 127) : (int)m;
				}
				held += s1 ? 1u : 0u;
			}
			c = pack4(lc[0], lc[1], lc[2], lc[3]);
		}
		// rotation
		const uint32_t other = a.halves ? __shfl_sync(0xffffffffu, c, e < a.rotary ? (e < a.rotary / 2 ? lane + half_lanes : lane - half_lanes) : lane) : 0u;
		if ((is_q || is_k) && e < a.rotary) {
			const int64_t row = (int64_t)pos * (a.rotary >> 1);
			if (!a.halves) {
				c = rope_quad(c, *(const int2*)(a.cos + row + (e >> 1)), *(const int2*)(a.sin + row + (e >> 1)));
			} else {
				const bool low = e < a.rotary / 2;
				const int at = low ? e : e - a.rotary / 2;
				const int4 cs = *(const int4*)(a.cos + row + at), sn = *(const int4*)(a.sin + row + at);
				const int co[4] = {cs.x, cs.y, cs.z, cs.w}, si[4] = {sn.x, sn.y, sn.z, sn.w};
				int out[4];
#pragma unroll
				for (int j = 0; j < 4; ++j) {
					const int mine = byte_of(c, j), theirs = byte_of(other, j);
					out[j] = rope_round(low ? (int64_t)mine * co[j] - (int64_t)theirs * si[j] : (int64_t)theirs * si[j] + (int64_t)mine * co[j]);
				}
				c = pack4(out[0], out[1], out[2], out[3]);
			}
		}
		if (is_q) {
			*(uint32_t*)(a.q_codes + r * a.q_codes_stride + 4 * i) = c;
		} else if (is_k) {
			*(uint32_t*)(a.kv + ((2 * (int64_t)head * a.num_pages + page) * kPageTokens + slot) * hd + e) = c;
		} else if (is_v) {
			int8_t* to = a.kv + (((2 * (int64_t)head + 1) * a.num_pages + page) * hd + e) * kPageTokens + slot;
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
		if (a.consts != nullptr) {
			for (int h = lane; h < a.kv_heads; h += 32) {
				const Scale kh{a.khead[2 * h], a.khead[2 * h + 1]};
				SoftmaxConsts sc;
				const bool none = softmax_consts(fp.out, kh, 1, &sc) != kOk;
				int64_t* to = a.consts + (r * a.kv_heads + h) * 3;
				to[0] = none ? 0 : sc.c.q_ln2;
				to[1] = none ? 0 : sc.c.q_b;
				to[2] = none ? 0 : sc.c.q_c;
				bad = bad || none;
			}
		}
	}
	bad = __any_sync(0xffffffffu, bad);
	if (lane == 0 && a.row_status != nullptr) a.row_status[r] = bad ? SSLM_B200_ROW_SOFTMAX : 0;
}

template <int NV>
cudaError_t site_launch(const SiteArgs& g, cudaStream_t st) {
	const int threads = ((g.total + NV - 1) / NV + 31) & ~31;
	return launch_pdl(k_qkv_site<NV>, dim3(g.c.rows), dim3(threads), 0, st, g);
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
	const cudaStream_t st = (cudaStream_t)stream;
	const cudaError_t e = g.total > 4096 ? site_launch<16>(g, st) : (g.total > 1024 || c.rows >= 512 ? site_launch<4>(g, st) : site_launch<1>(g, st));
	if (e != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}
