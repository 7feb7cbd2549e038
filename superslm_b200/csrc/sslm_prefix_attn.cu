// Integer i-exp softmax attention of rows that share a prefix, the prefix computed once for all of them.
//
// Rows (one token of one sequence each) come in groups; the rows of a group see the same P positions and
// then S_r of their own. The arithmetic of a row is that of k_attention (sslm_attn.cu), over P + S_r positions:
//   s_k = q . K_k,  e_k = i-exp(s_k - max),  p_k = floor(2^15 e_k / sum),  ctx = sum p_k V_k,  fold
// A tile is ROWS query rows of one kv head: tq = ROWS / G rows of a group times the G q heads of that kv head.
// The tile multiplies the prefix's K and V once, ROWS rows at a time; a row's own pages are multiplied
// with the same instructions, the other rows of the tile left out. A tile is cut over the blocks of a
// cluster, prefix in steps of 128 positions and suffixes in pages of 16, both dealt round-robin, and the
// blocks exchange maxima, sums and shares of P.V as k_attention_chunk's do (sums and maxima of integers:
// no order of arrival changes a result).
//
// The scores of a step lie in shared memory, four neighbouring positions of a row per word quad: of the
// prefix where the thread that computed them finds them again, of suffix pages packed by (page, head), since
// only G of the tile's rows see such a page. Both become the A fragments of P.V in place.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/sslm_b200.h"
#include "sslm_cluster.cuh"
#include "sslm_kernels.h"
#include "sslm_quad.cuh"
#include "sslm_softmax.cuh"

namespace sslm {

constexpr int kPfxThreads = 256, kPfxStep = 128, kPfxStepPages = kPfxStep / kPageTokens;
constexpr int kPfxMaxWidth = 32768;      // positions a row sees at most: the longest admitted context
constexpr int kPfxTokens = 32;           // rows a tile holds at most (32 query rows of groups of one)

struct PrefixArgs {
	int rows, groups, G, kv_heads, tq, ginv, shift;      // ginv = ceil(65536 / G); a tile is cut over 1 << shift blocks
	int psteps, spages;                                  // prefix steps and suffix pages a block has room for
	int max_prefix, max_suffix;
	const int8_t* q;
	int64_t q_stride;
	const int8_t* kv;              // [kv_heads][K|V] planes of num_pages pages
	int64_t num_pages;
	const int32_t *group_start, *prefix_len;
	// a caller's tensors
	const int64_t* consts;         // [rows][kv_heads][3]
	const int32_t *prefix_pages, *suffix_len, *suffix_pages;
	int64_t prefix_stride, suffix_stride;
	// rows of an engine call
	const RowDesc* desc;
	const SoftmaxConsts* smc;      // [rows][kv_heads]
	unsigned long long* rowmax;    // [rows][4], slot 3
	int layer;
	const int32_t* fold;           // [heads][3], or nullptr: none
	int32_t* out;
	int64_t out_stride;
	int32_t* status;
	int debug_withhold;            // tests only (exchange_debug_take)
};

template <int HD, int ROWS>
struct PrefixSmem {
	static constexpr int kKStride = HD + 16;                                        // (padding against bank conflicts)
	static constexpr size_t kStage = (size_t)2 * kPfxStep * kKStride;               // two K steps, two V steps, or received shares
	static constexpr size_t kStepScores = (size_t)ROWS * kPfxStep * 4;
	static constexpr size_t bytes(int psteps, int spages, int group) {
		return kStage + kStepScores * psteps + (size_t)spages * group * kPageTokens * 4 + (size_t)(psteps * kPfxStepPages + spages) * 8 + (size_t)spages * 4;
	}
};

// the constants of a row's softmax element lie where the kernels' short forms hold, and a row of `width` such
// elements adds up in 63 bits (the gates of the q/k/v site)
__device__ __forceinline__ bool softmax_gate(int64_t ln2, int64_t qb, int64_t qc, int width) {
	if (ln2 < 1 || ln2 > qb || qb >= (1 << 24) || qc < 0 || qc > SSLM_SOFTMAX_MAX_SAFE) return false;
	const int64_t peak = qb * qb + qc;      // (below 2^49)
	return peak <= SSLM_SOFTMAX_MAX_SAFE && (unsigned long long)peak * (unsigned long long)max(width, 1) <= 0x7FFFFFFFFFFFFFFFull;
}

template <int HD, int ROWS, bool RESIDENT>
__global__ void __launch_bounds__(kPfxThreads, 2) k_attention_prefix(const __grid_constant__ PrefixArgs a) {
	using L = PrefixSmem<HD, ROWS>;
	constexpr int KS = HD / 32;                       // MMA steps along the head dimension
	constexpr int RB = ROWS / 16;                     // 16-row blocks
	constexpr int CW = 8 / RB;                        // warps per row block: along the pages of a step, along the channels of P.V
	constexpr int PW = kPfxStepPages / CW;            // pages of a step per warp
	constexpr int NT = HD / 8 >= CW ? HD / 8 / CW : 1;      // 8-channel tiles a warp owns in P.V (some warps none: 32 channels, 16 rows)
	constexpr int kSlots = RB * 32;
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ __align__(8) unsigned long long s_bars[3];
	__shared__ unsigned long long s_sum[ROWS], s_rxsum[kPfxThreads];
	__shared__ IExpFast s_fx[kPfxTokens];
	__shared__ int32_t s_max[ROWS], s_rxmax[kPfxThreads], s_len[kPfxTokens], s_code[kPfxTokens], s_cum[kPfxTokens + 1], s_fold[24], s_tile[3], s_badprefix;

	const int G = a.G, kvh = (int)blockIdx.z;
	const int sub = 1 << a.shift, rank = (int)blockIdx.x;
	const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, c = lane & 3;
	int8_t* stage = (int8_t*)smem;
	int4* sc = (int4*)(smem + L::kStage);                                                       // [step][page][row a, row b][kSlots]
	int4* csc = (int4*)(smem + L::kStage + L::kStepScores * a.psteps);                          // [suffix page][head][4]
	int64_t* pbase = (int64_t*)((unsigned char*)csc + (size_t)a.spages * G * kPageTokens * 4);  // page offsets inside a plane, -1: none
	int64_t* sbase = pbase + a.psteps * kPfxStepPages;
	int32_t* sown = (int32_t*)(sbase + a.spages);                                               // owner | positions << 8
	int32_t* rx_ctx = (int32_t*)stage;                                                          // [sub][ROWS / sub][HD]

	if (sub > 1) {
		if (t == 0) {
			const int held = (blockIdx.x | blockIdx.y | blockIdx.z) == 0 ? a.debug_withhold : 0;
			auto more = [&](int i) { return held == i + 1 ? 4u : 0u; };
			exchange_init(cta_addr(&s_bars[0]), (uint32_t)(sub * ROWS * 4) + more(0));
			exchange_init(cta_addr(&s_bars[1]), (uint32_t)(sub * ROWS * 8) + more(1));
			exchange_init(cta_addr(&s_bars[2]), (uint32_t)(ROWS * HD * 4) + more(2));
			exchange_fence_init();
		}
		cluster_arrive();
		cluster_wait();
	}
	// A caller's tensors may have been written by the kernel in front. An engine call's descriptors, lengths and page
	// tables were uploaded, and the prefix's pages filled, before its first launch.
	if (RESIDENT) {
		pdl_wait();
		pdl_release();
	}
	// ---- which tile: group after group, tq rows at a time
	if (warp == 0) {
		int want = (int)blockIdx.y, r0 = 0, nt = 0, group = 0;
		for (int g0 = 0; g0 < a.groups; g0 += 32) {
			int start = 0, n = 0;
			if (g0 + lane < a.groups) {
				start = max(a.group_start[g0 + lane], 0);
				n = max(min(a.group_start[g0 + lane + 1], a.rows) - start, 0);
			}
			const int tiles = (n + a.tq - 1) / a.tq;
			int upto = tiles;
#pragma unroll
			for (int o = 1; o < 32; o *= 2) {
				const int v = __shfl_up_sync(0xffffffffu, upto, o);
				if (lane >= o) upto += v;
			}
			const uint32_t has = __ballot_sync(0xffffffffu, want < upto);
			if (has != 0u) {
				const int src = __ffs(has) - 1, first = (want - (upto - tiles)) * a.tq;
				r0 = __shfl_sync(0xffffffffu, start + first, src);
				nt = __shfl_sync(0xffffffffu, min(a.tq, n - first), src);
				group = g0 + src;
				break;
			}
			want -= __shfl_sync(0xffffffffu, upto, 31);
		}
		if (lane == 0) {
			s_tile[0] = r0;
			s_tile[1] = nt;
			s_tile[2] = group;
			s_badprefix = 0;
		}
	}
	if (t < ROWS) {
		s_max[t] = INT32_MIN;
		s_sum[t] = 0ull;
	}
	if (t < 3 * G) s_fold[t] = a.fold != nullptr ? a.fold[3 * kvh * G + t] : (t % 3 == 0 ? 1 : 0);
	__syncthreads();
	const int r0 = s_tile[0], nt = s_tile[1], group = s_tile[2];
	if (nt == 0) return;      // (all blocks of the cluster alike)
	int P = a.prefix_len[group];
	const int32_t* prefix_pages = RESIDENT ? a.prefix_pages + (int64_t)group * a.prefix_stride : a.desc[r0].pages;
	if (RESIDENT) {
		// lengths, constants and page ids that are out of range refuse their row; every block of the tile comes to the
		// same verdict by itself
		const bool bad_len = P < 0 || P > a.max_prefix;
		if (t < kPfxTokens) {
			int code = kOk, len = 0;
			if (t < nt) {
				len = a.suffix_len[r0 + t];
				if (bad_len || len < 0 || len > a.max_suffix || P + len > kPfxMaxWidth) {
					code = SSLM_B200_ROW_LENGTH;
				} else {
					const int64_t* k = a.consts + (int64_t)(r0 + t) * a.kv_heads * 3;
					for (int h = 0; h < a.kv_heads; ++h)
						if (!softmax_gate(k[3 * h], k[3 * h + 1], k[3 * h + 2], P + len)) code = SSLM_B200_ROW_CONSTANTS;
				}
			}
			s_len[t] = code == kOk ? len : 0;
			s_code[t] = code;
		}
		if (bad_len) P = 0;
		__syncthreads();
		for (int i = t; i < (P + kPageTokens - 1) / kPageTokens; i += kPfxThreads)
			if ((uint64_t)(int64_t)prefix_pages[i] >= (uint64_t)a.num_pages) s_badprefix = 1;
		for (int tk = warp; tk < nt; tk += kPfxThreads / 32) {
			const int32_t* pages = a.suffix_pages + (int64_t)(r0 + tk) * a.suffix_stride;
			bool bad = false;
			for (int i = lane; i < (s_len[tk] + kPageTokens - 1) / kPageTokens; i += 32) bad = bad || (uint64_t)(int64_t)pages[i] >= (uint64_t)a.num_pages;
			if (__any_sync(0xffffffffu, bad) && lane == 0) {
				s_code[tk] = SSLM_B200_ROW_INDEX;
				s_len[tk] = 0;
			}
		}
		__syncthreads();
		if (s_badprefix != 0) {
			P = 0;
			if (t < nt && s_code[t] == kOk) s_code[t] = SSLM_B200_ROW_INDEX;
			if (t < kPfxTokens) s_len[t] = 0;
			__syncthreads();
		}
		// (the tiles of the first kv head start first: what a later one may have to say about a wait comes after this)
		if (kvh == 0 && rank == 0 && t < nt && a.status != nullptr) a.status[r0 + t] = s_code[t];
	} else if (t < kPfxTokens) {
		s_len[t] = t < nt ? min(max(a.desc[r0 + t].pos + 1 - P, 0), a.max_suffix) : 0;
	}
	if (warp == 0) {      // pages of the tile's suffixes, counted up row by row
		__syncwarp();
		int upto = (s_len[lane] + kPageTokens - 1) / kPageTokens;
#pragma unroll
		for (int o = 1; o < 32; o *= 2) {
			const int v = __shfl_up_sync(0xffffffffu, upto, o);
			if (lane >= o) upto += v;
		}
		s_cum[lane + 1] = upto;
		if (lane == 0) s_cum[0] = 0;
	}
	__syncthreads();
	// ---- this block's part: prefix steps and suffix pages rank, rank + sub, ...
	auto mine = [&](int n) { return n > rank ? (n - rank + sub - 1) >> a.shift : 0; };
	const int nps = min(mine((P + kPfxStep - 1) / kPfxStep), a.psteps);
	const int nsp = min(mine(s_cum[kPfxTokens]), a.spages);
	const int nss = (nsp + kPfxStepPages - 1) / kPfxStepPages, steps = nps + nss;
	const int64_t page_bytes = kPageTokens * HD, plane = a.num_pages * page_bytes;
	const int8_t* kplane = a.kv + (int64_t)(2 * kvh) * plane;
	const int8_t* vplane = kplane + plane;
	for (int i = t; i < nps * kPfxStepPages; i += kPfxThreads) {
		const int page = (rank + (i / kPfxStepPages) * sub) * kPfxStepPages + i % kPfxStepPages;
		pbase[i] = page * kPageTokens < P ? (int64_t)prefix_pages[page] * page_bytes : -1;
	}
	for (int i = t; i < nss * kPfxStepPages; i += kPfxThreads) {
		int64_t base = -1;
		int own = 255;
		if (i < nsp) {
			const int x = rank + i * sub;
			int tk = 0;
			while (s_cum[tk + 1] <= x) ++tk;
			const int page = x - s_cum[tk];
			const int32_t* pages = RESIDENT ? a.suffix_pages + (int64_t)(r0 + tk) * a.suffix_stride : a.desc[r0 + tk].pages + P / kPageTokens;
			base = (int64_t)pages[page] * page_bytes;
			own = tk | min(kPageTokens, s_len[tk] - page * kPageTokens) << 8;
		}
		sbase[i] = base;
		sown[i] = own;
	}
	__syncthreads();
	// step i into half i & 1 of the stage; pages that there are not are left out (their scores are masked, their
	// probabilities zero)
	auto base_of = [&](int i, int page) { return i < nps ? pbase[i * kPfxStepPages + page] : sbase[(i - nps) * kPfxStepPages + page]; };
	auto load_k = [&](int i) {
		int8_t* kd = stage + (size_t)(i & 1) * kPfxStep * L::kKStride;
		for (int idx = t; idx < kPfxStep * (HD / 16); idx += kPfxThreads) {
			const int row = idx / (HD / 16), piece = idx % (HD / 16);
			const int64_t base = base_of(i, row / kPageTokens);
			if (base >= 0) cp_async16(kd + (size_t)row * L::kKStride + piece * 16, kplane + base + (row % kPageTokens) * HD + piece * 16);
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	auto load_v = [&](int i) {
		int8_t* vd = stage + (size_t)(i & 1) * kPfxStep * HD;
		for (int idx = t; idx < kPfxStepPages * HD; idx += kPfxThreads) {
			const int pg = idx / HD, piece = idx % HD;
			const int64_t base = base_of(i, pg);
			if (base >= 0) cp_async16(vd + (size_t)pg * HD * kPageTokens + piece * 16, vplane + base + piece * 16);
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	const bool early = RESIDENT || nps > 0;      // (an engine call's newest K rows come from the kernel in front)
	if (early && steps > 0) load_k(0);
	if (!RESIDENT) {
		pdl_wait();
		pdl_release();
	}
	if (!early && steps > 0) load_k(0);
	if (t < kPfxTokens) {
		IExpFast f{1u, 30u, 1, 0, 0.9999995f};
		if (t < nt) {
			if (RESIDENT) {
				const int64_t* k = a.consts + ((int64_t)(r0 + t) * a.kv_heads + kvh) * 3;
				if (s_code[t] == kOk) f = iexp_fast_prepare(SoftmaxConsts{{k[0], k[1], k[2]}, 0});
			} else {
				s_code[t] = __ldcg(&a.status[r0 + t]) != 0 ? 1 : kOk;
				if (s_code[t] == kOk) f = iexp_fast_prepare(a.smc[(size_t)(r0 + t) * a.kv_heads + kvh]);
			}
		} else {
			s_code[t] = 1;
		}
		s_fx[t] = f;
	}
	__syncthreads();

	const int rb = warp / CW, kq = warp % CW;
	const int rho_a = rb * 16 + g, rho_b = rho_a + 8;
	const int tok_a = rho_a * a.ginv >> 16, tok_b = rho_b * a.ginv >> 16;
	const int head_a = rho_a - tok_a * G, head_b = rho_b - tok_b * G;
	const bool in_a = tok_a < nt && s_code[tok_a] == kOk, in_b = tok_b < nt && s_code[tok_b] == kOk;
	bool ok = true;

	// ---- pass 1: scores and row maxima. acc[j]: MMA j = 2 * page + half; the K rows of a page are read in the order
	// 0 1 4 5 8 9 12 13 | 2 3 6 7 10 11 14 15, which leaves a lane with four neighbouring positions
	{
		uint32_t qa[KS][4];
		const int8_t* qpa = a.q + (int64_t)(r0 + (in_a ? tok_a : 0)) * a.q_stride + (int64_t)(kvh * G + head_a) * HD;
		const int8_t* qpb = a.q + (int64_t)(r0 + (in_b ? tok_b : 0)) * a.q_stride + (int64_t)(kvh * G + head_b) * HD;
#pragma unroll
		for (int ks = 0; ks < KS; ++ks) {
			qa[ks][0] = in_a ? *(const uint32_t*)(qpa + 32 * ks + 4 * c) : 0u;
			qa[ks][1] = in_b ? *(const uint32_t*)(qpb + 32 * ks + 4 * c) : 0u;
			qa[ks][2] = in_a ? *(const uint32_t*)(qpa + 32 * ks + 16 + 4 * c) : 0u;
			qa[ks][3] = in_b ? *(const uint32_t*)(qpb + 32 * ks + 16 + 4 * c) : 0u;
		}
		const int krow = 4 * ((lane & 7) >> 1) + (lane & 1);
		int mx_a = INT32_MIN, mx_b = INT32_MIN;
#pragma unroll 1
		for (int i = 0; i < steps; ++i) {
			if (i + 1 < steps) {
				load_k(i + 1);
				asm volatile("cp.async.wait_group 1;" ::: "memory");
			} else {
				asm volatile("cp.async.wait_group 0;" ::: "memory");
			}
			__syncthreads();
			const uint32_t kd = cta_addr(stage + (size_t)((i & 1) * kPfxStep + kq * PW * kPageTokens) * L::kKStride);
			int acc[2 * PW][4];
#pragma unroll
			for (int j = 0; j < 2 * PW; ++j)
#pragma unroll
				for (int x = 0; x < 4; ++x) acc[j][x] = 0;
			if constexpr (HD == 32) {
#pragma unroll
				for (int j = 0; j < 2 * PW; j += 2) {      // both halves of a page in one load
					uint32_t b0, b1, b2, b3;
					ldmatrix4(kd + (8 * j + krow + 2 * (lane >> 4)) * L::kKStride + ((lane >> 3) & 1) * 16, b0, b1, b2, b3);
					mma_s8s8_full(acc[j], qa[0][0], qa[0][1], qa[0][2], qa[0][3], b0, b1);
					mma_s8s8_full(acc[j + 1], qa[0][0], qa[0][1], qa[0][2], qa[0][3], b2, b3);
				}
			} else {
#pragma unroll
				for (int ks = 0; ks < KS; ks += 2) {
#pragma unroll
					for (int j = 0; j < 2 * PW; ++j) {
						uint32_t b0, b1, b2, b3;
						ldmatrix4(kd + (16 * (j >> 1) + 2 * (j & 1) + krow) * L::kKStride + 32 * ks + (lane >> 3) * 16, b0, b1, b2, b3);
						mma_s8s8_full(acc[j], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b0, b1);
						mma_s8s8_full(acc[j], qa[ks + 1][0], qa[ks + 1][1], qa[ks + 1][2], qa[ks + 1][3], b2, b3);
					}
				}
			}
			// row a, page p (positions 4 c ..): acc[2p][0], acc[2p][1], acc[2p + 1][0], acc[2p + 1][1]; row b: [2], [3]
#pragma unroll
			for (int p = 0; p < PW; ++p) {
				int4 va = make_int4(acc[2 * p][0], acc[2 * p][1], acc[2 * p + 1][0], acc[2 * p + 1][1]);
				int4 vb = make_int4(acc[2 * p][2], acc[2 * p][3], acc[2 * p + 1][2], acc[2 * p + 1][3]);
				const int page = kq * PW + p;
				bool see_a = true, see_b = true;
				int end;      // positions of the page that count
				if (i < nps) {
					end = P - ((rank + i * sub) * kPfxStep + page * kPageTokens);
				} else {
					const int own = sown[(i - nps) * kPfxStepPages + page];
					end = own >> 8;
					see_a = tok_a == (own & 255);
					see_b = tok_b == (own & 255);
				}
				if (end < kPageTokens) {
					const int k0 = 4 * c;
					va.x = k0 < end ? va.x : INT32_MIN; va.y = k0 + 1 < end ? va.y : INT32_MIN;
					va.z = k0 + 2 < end ? va.z : INT32_MIN; va.w = k0 + 3 < end ? va.w : INT32_MIN;
					vb.x = k0 < end ? vb.x : INT32_MIN; vb.y = k0 + 1 < end ? vb.y : INT32_MIN;
					vb.z = k0 + 2 < end ? vb.z : INT32_MIN; vb.w = k0 + 3 < end ? vb.w : INT32_MIN;
				}
				if (see_a) mx_a = max(mx_a, max(max(va.x, va.y), max(va.z, va.w)));
				if (see_b) mx_b = max(mx_b, max(max(vb.x, vb.y), max(vb.z, vb.w)));
				if (i < nps) {
					int4* at = sc + ((size_t)(i * kPfxStepPages + page) * 2) * kSlots + rb * 32 + lane;
					at[0] = va;
					at[kSlots] = vb;
				} else {
					int4* at = csc + (size_t)((i - nps) * kPfxStepPages + page) * G * 4 + c;
					if (see_a) at[4 * head_a] = va;
					if (see_b) at[4 * head_b] = vb;
				}
			}
			__syncthreads();      // the step may be overwritten
		}
		mx_a = max(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1));
		mx_a = max(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
		mx_b = max(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1));
		mx_b = max(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
		if (c == 0) {
			atomicMax(&s_max[rho_a], mx_a);
			atomicMax(&s_max[rho_b], mx_b);
		}
	}
	// (the stage is free: V arrives during the softmax)
	if (steps > 0) load_v(0);
	if (steps > 1) load_v(1);
	__syncthreads();
	if (sub > 1) {
		if (t < sub * ROWS) exchange_send(&s_rxmax[rank * ROWS + t % ROWS], cta_addr(&s_bars[0]), (uint32_t)(t / ROWS), (uint32_t)s_max[t % ROWS]);
		ok = exchange_wait(cta_addr(&s_bars[0]));
		__syncthreads();
		if (t < ROWS) {
			int m = INT32_MIN;
			for (int i = 0; i < sub; ++i) m = max(m, s_rxmax[i * ROWS + t]);
			s_max[t] = m;
		}
		__syncthreads();
	}

	// ---- pass 2: exponentials and row totals; a score's place then holds the element's (shift, base)
	const IExpFast fa = s_fx[in_a ? tok_a : 0], fb = s_fx[in_b ? tok_b : 0];
	const int ntask = nsp * G * 4;      // four positions of one head and suffix page each
	{
		const uint32_t mx_a = (uint32_t)s_max[rho_a], mx_b = (uint32_t)s_max[rho_b];
		unsigned long long sum[2] = {0ull, 0ull};
		auto four = [](int4 v, uint32_t m, const IExpFast& f, bool whole, int4* parts) {
			uint32_t p0, p1, p2, p3;
			int64_t e0 = chunk_exp(m - (uint32_t)v.x, f, &p0), e1 = chunk_exp(m - (uint32_t)v.y, f, &p1);
			int64_t e2 = chunk_exp(m - (uint32_t)v.z, f, &p2), e3 = chunk_exp(m - (uint32_t)v.w, f, &p3);
			if (!whole) {      // masked positions count for nothing
				if (v.x == INT32_MIN) { e0 = 0; p0 = kBaseOfZero; }
				if (v.y == INT32_MIN) { e1 = 0; p1 = kBaseOfZero; }
				if (v.z == INT32_MIN) { e2 = 0; p2 = kBaseOfZero; }
				if (v.w == INT32_MIN) { e3 = 0; p3 = kBaseOfZero; }
			}
			*parts = make_int4((int)p0, (int)p1, (int)p2, (int)p3);
			return (unsigned long long)(e0 + e1) + (unsigned long long)(e2 + e3);
		};
#pragma unroll 1
		for (int i = 0; i < nps; ++i) {
			const bool whole = (rank + i * sub) * kPfxStep + kPfxStep <= P;
#pragma unroll
			for (int p = 0; p < PW; ++p) {
				int4* at = sc + ((size_t)(i * kPfxStepPages + kq * PW + p) * 2) * kSlots + rb * 32 + lane;
				sum[0] += four(at[0], mx_a, fa, whole, &at[0]);
				sum[1] += four(at[kSlots], mx_b, fb, whole, &at[kSlots]);
			}
		}
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
			sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
			if (c == 0 && nps > 0) atomicAdd(&s_sum[h ? rho_b : rho_a], sum[h]);
		}
#pragma unroll 1
		for (int u0 = warp * 32; u0 < ntask; u0 += kPfxThreads) {
			const int u = u0 + lane;
			unsigned long long s = 0ull;
			int rho = 0;
			if (u < ntask) {
				const int page = (u >> 2) * a.ginv >> 16, head = (u >> 2) - page * G, own = sown[page];
				rho = (own & 255) * G + head;
				s = four(csc[u], (uint32_t)s_max[rho], s_fx[own & 255], own >> 8 == kPageTokens, &csc[u]);
			}
			s += __shfl_xor_sync(0xffffffffu, s, 1);
			s += __shfl_xor_sync(0xffffffffu, s, 2);
			if (c == 0 && u < ntask) atomicAdd(&s_sum[rho], s);
		}
	}
	__syncthreads();
	if (sub > 1) {
		if (t < sub * ROWS) exchange_send(&s_rxsum[rank * ROWS + t % ROWS], cta_addr(&s_bars[1]), (uint32_t)(t / ROWS), s_sum[t % ROWS]);
		ok = exchange_wait(cta_addr(&s_bars[1])) && ok;
		__syncthreads();
		if (t < ROWS) {
			unsigned long long s = 0ull;
			for (int i = 0; i < sub; ++i) s += s_rxsum[i * ROWS + t];
			s_sum[t] = s;
		}
		__syncthreads();
	}

	// ---- pass 3: probabilities, packed as the A fragments of P.V: of a prefix page (row a low, row b low, row a high, row b
	// high plane), of a suffix page and head (low, high), four positions per word
	{
		auto four = [](int4 v, const ChunkProb& p, int64_t qc, unsigned long long tot, uint32_t* lo, uint32_t* hi) {
			float near = 1.0f;
			uint32_t p0 = chunk_prob_of((uint32_t)v.x, p, &near), p1 = chunk_prob_of((uint32_t)v.y, p, &near);
			uint32_t p2 = chunk_prob_of((uint32_t)v.z, p, &near), p3 = chunk_prob_of((uint32_t)v.w, p, &near);
			if (near < p.eps) {
				const uint4 x = chunk_prob_exact((uint32_t)v.x, (uint32_t)v.y, (uint32_t)v.z, (uint32_t)v.w, qc, tot);
				p0 = x.x; p1 = x.y; p2 = x.z; p3 = x.w;
			}
			*lo = pack_plane(p0, p1, p2, p3, 0);
			*hi = pack_plane(p0, p1, p2, p3, 1);
		};
		const unsigned long long tot_a = s_sum[rho_a], tot_b = s_sum[rho_b];
		const ChunkProb pa = chunk_prob(tot_a, fa), pb = chunk_prob(tot_b, fb);
#pragma unroll 1
		for (int i = 0; i < nps; ++i) {
#pragma unroll
			for (int p = 0; p < PW; ++p) {
				int4* at = sc + ((size_t)(i * kPfxStepPages + kq * PW + p) * 2) * kSlots + rb * 32 + lane;
				uint32_t lo_a, hi_a, lo_b, hi_b;
				four(at[0], pa, fa.qc, tot_a, &lo_a, &hi_a);
				four(at[kSlots], pb, fb.qc, tot_b, &lo_b, &hi_b);
				at[0] = make_int4((int)lo_a, (int)lo_b, (int)hi_a, (int)hi_b);
			}
		}
#pragma unroll 1
		for (int u = t; u < ntask; u += kPfxThreads) {
			const int page = (u >> 2) * a.ginv >> 16, head = (u >> 2) - page * G, tk = sown[page] & 255;
			const unsigned long long tot = s_sum[tk * G + head];
			uint32_t lo, hi;
			four(csc[u], chunk_prob(tot, s_fx[tk]), s_fx[tk].qc, tot, &lo, &hi);
			csc[u] = make_int4((int)lo, (int)hi, 0, 0);
		}
	}

	// ---- pass 4: P.V of this warp's rows and channels, over the pages of all warps
	const bool owns = kq * NT * 8 < HD;
	int accl[NT][4], acch[NT][4];
#pragma unroll
	for (int i = 0; i < NT; ++i)
#pragma unroll
		for (int x = 0; x < 4; ++x) accl[i][x] = acch[i][x] = 0;
#pragma unroll 1
	for (int i = 0; i < steps; ++i) {
		if (i + 1 < steps) asm volatile("cp.async.wait_group 1;" ::: "memory");
		else asm volatile("cp.async.wait_group 0;" ::: "memory");
		__syncthreads();      // V of the step (and, the first time, everybody's probabilities) are there
		const uint32_t vd = cta_addr(stage + (size_t)(i & 1) * kPfxStep * HD);
		if (owns) {
#pragma unroll
			for (int ks = 0; ks < kPfxStepPages / 2; ++ks) {      // two pages
				int4 x0, x1;
				if (i < nps) {
					const int4* at = sc + ((size_t)(i * kPfxStepPages + 2 * ks) * 2) * kSlots + rb * 32 + lane;
					x0 = at[0];
					x1 = at[2 * kSlots];
				} else {
					const int page = (i - nps) * kPfxStepPages + 2 * ks;
					auto fragment = [&](int pg) {
						const int own = sown[pg] & 255;
						int2 fa2 = make_int2(0, 0), fb2 = make_int2(0, 0);
						if (tok_a == own) fa2 = *(const int2*)&csc[(size_t)(pg * G + head_a) * 4 + c];
						if (tok_b == own) fb2 = *(const int2*)&csc[(size_t)(pg * G + head_b) * 4 + c];
						return make_int4(fa2.x, fb2.x, fa2.y, fb2.y);
					};
					x0 = fragment(page);
					x1 = fragment(page + 1);
				}
				if constexpr (NT == 1) {
					const uint32_t at = vd + (uint32_t)((2 * ks + ((lane >> 3) & 1)) * HD + 8 * kq + (lane & 7)) * kPageTokens;
					uint32_t b0, b1, b2, b3;      // (the upper half of the lanes repeats the lower half's rows)
					ldmatrix4(at, b0, b1, b2, b3);
					mma_u8s8_full(accl[0], x0.x, x0.y, x1.x, x1.y, b0, b1);
					mma_u8s8_full(acch[0], x0.z, x0.w, x1.z, x1.w, b0, b1);
				} else {
#pragma unroll
					for (int n = 0; n < NT; n += 2) {      // two 8-channel tiles, two pages each
						const uint32_t at = vd + (uint32_t)((2 * ks + ((lane >> 3) & 1)) * HD + 8 * (kq * NT + n + (lane >> 4)) + (lane & 7)) * kPageTokens;
						uint32_t b0, b1, b2, b3;
						ldmatrix4(at, b0, b1, b2, b3);
						mma_u8s8_full(accl[n], x0.x, x0.y, x1.x, x1.y, b0, b1);
						mma_u8s8_full(acch[n], x0.z, x0.w, x1.z, x1.w, b0, b1);
						mma_u8s8_full(accl[n + 1], x0.x, x0.y, x1.x, x1.y, b2, b3);
						mma_u8s8_full(acch[n + 1], x0.z, x0.w, x1.z, x1.w, b2, b3);
					}
				}
			}
		}
		__syncthreads();      // the step may be overwritten
		if (i + 2 < steps) load_v(i + 2);
	}

	// ---- per-head context fold (forward_sites.cpp:1889-1896), store, row maximum for the funnel
	if (sub == 1) {
		uint32_t top_a = 0, top_b = 0;
		if (owns) {
#pragma unroll
			for (int n = 0; n < NT; ++n) {
				const int ch = 8 * (kq * NT + n) + 2 * c;
				auto put = [&](int tok, int head, int v0, int v1, uint32_t& top) {
					int2 o;
					o.x = fold(v0, s_fold[3 * head], s_fold[3 * head + 1], s_fold[3 * head + 2]);
					o.y = fold(v1, s_fold[3 * head], s_fold[3 * head + 1], s_fold[3 * head + 2]);
					*(int2*)(a.out + (int64_t)(r0 + tok) * a.out_stride + (int64_t)(kvh * G + head) * HD + ch) = o;
					top = max(top, max(abs_u32(o.x), abs_u32(o.y)));
				};
				if (in_a) put(tok_a, head_a, accl[n][0] + 256 * acch[n][0], accl[n][1] + 256 * acch[n][1], top_a);
				if (in_b) put(tok_b, head_b, accl[n][2] + 256 * acch[n][2], accl[n][3] + 256 * acch[n][3], top_b);
			}
		}
		if (!RESIDENT) {
			top_a = max(top_a, __shfl_xor_sync(0xffffffffu, top_a, 1));
			top_a = max(top_a, __shfl_xor_sync(0xffffffffu, top_a, 2));
			top_b = max(top_b, __shfl_xor_sync(0xffffffffu, top_b, 1));
			top_b = max(top_b, __shfl_xor_sync(0xffffffffu, top_b, 2));
			if (c == 0 && top_a) atomicMax(&a.rowmax[(size_t)(r0 + tok_a) * 4 + 3], (unsigned long long)top_a);
			if (c == 0 && top_b) atomicMax(&a.rowmax[(size_t)(r0 + tok_b) * 4 + 3], (unsigned long long)top_b);
		}
		return;
	}
	// the shares go to the blocks that add them up; a peer's stage is free once the peer has got here
	cluster_arrive();
	cluster_wait();
	constexpr int kRowBits = ROWS == 32 ? 5 : 4;
	const int rows = ROWS >> a.shift, rshift = kRowBits - a.shift;
	auto send = [&](int rho, int ch, int v0, int v1) {
		exchange_send(&rx_ctx[(rank * rows + (rho & (rows - 1))) * HD + ch], cta_addr(&s_bars[2]), (uint32_t)(rho >> rshift), make_int2(v0, v1));
	};
	if (owns) {
#pragma unroll
		for (int n = 0; n < NT; ++n) {
			const int ch = 8 * (kq * NT + n) + 2 * c;
			send(rho_a, ch, accl[n][0] + 256 * acch[n][0], accl[n][1] + 256 * acch[n][1]);
			send(rho_b, ch, accl[n][2] + 256 * acch[n][2], accl[n][3] + 256 * acch[n][3]);
		}
	}
	ok = exchange_wait(cta_addr(&s_bars[2])) && ok;
	for (int e = t; e < rows * HD; e += kPfxThreads) {
		const int rho = rank * rows + e / HD, ch = e % HD, tok = rho * a.ginv >> 16, head = rho - tok * G;      // (a warp's elements lie in one row)
		int32_t sum = 0;
		for (int i = 0; i < sub; ++i) sum += rx_ctx[i * rows * HD + e];
		const int32_t o = fold(sum, s_fold[3 * head], s_fold[3 * head + 1], s_fold[3 * head + 2]);
		const bool in = tok < nt && s_code[tok] == kOk;
		if (in) a.out[(int64_t)(r0 + tok) * a.out_stride + (int64_t)(kvh * G + head) * HD + ch] = o;
		if (!RESIDENT) {
			const uint32_t top = __reduce_max_sync(0xffffffffu, in ? abs_u32(o) : 0u);
			if (lane == 0 && top) atomicMax(&a.rowmax[(size_t)(r0 + tok) * 4 + 3], (unsigned long long)top);
		}
	}
	if (__builtin_expect(!__all_sync(0xffffffffu, ok), 0)) {      // (the warp's lanes speak for the tile's rows)
		if (lane < nt && a.status != nullptr) {
			if (RESIDENT) a.status[r0 + lane] = kInternalWaitTimeout;
			else atomicCAS(&a.status[r0 + lane], 0, pack_status(kInternalWaitTimeout, kSiteCtx, a.layer));
		}
		__syncwarp();
		exchange_leave(cta_addr(&s_bars[0]), 3);
	}
}

// Funnel of the context rows (forward_sites.cpp:1898-1903: no incoming scale, the site constant): codes and scale of every
// row of a group that was not refused. One block per row; the row's maximum is taken from the row itself.
__global__ void __launch_bounds__(256) k_prefix_codes(const int32_t* out, int64_t out_stride, int n, const int32_t* group_start, int groups, Scale site,
                                                      int8_t* codes, Scale* scales, int32_t* status) {
	__shared__ uint32_t s_top[8];
	const int r = blockIdx.x, t = threadIdx.x;
	const FunnelFold fold = funnel_prefold(nullptr, 0, site);
	pdl_wait();
	pdl_release();
	if (r < group_start[0] || r >= group_start[groups] || __ldcg(&status[r]) != 0) return;
	const int32_t* row = out + (int64_t)r * out_stride;
	uint32_t top = 0;
	for (int q = t; q < n / 4; q += 256) {
		int32_t x[4];
		load_quad(row + 4 * q, x);
#pragma unroll
		for (int j = 0; j < 4; ++j) top = max(top, abs_u32(x[j]));
	}
	top = __reduce_max_sync(0xffffffffu, top);
	if ((t & 31) == 0) s_top[t >> 5] = top;
	__syncthreads();
#pragma unroll
	for (int w = 0; w < 8; ++w) top = max(top, s_top[w]);
	const QuadFunnel fp = quad_funnel((unsigned long long)top, fold);
	if (t == 0) {
		if (fp.status != kOk) status[r] = fp.status;
		else if (scales != nullptr) scales[r] = fp.out;
	}
	if (fp.status != kOk) return;
	for (int q = t; q < n / 4; q += 256) {
		int32_t x[4];
		load_quad(row + 4 * q, x);
		((uint32_t*)(codes + (int64_t)r * n))[q] = code_quad(x, fp);
	}
}

namespace {

struct PrefixPlan {
	int rows;        // query rows per tile: 16 or 32
	int tq, tiles, shift, psteps, spages;
	size_t smem;
};
constexpr size_t kPfxSmemMax = 218 * 1024;      // (beside 9 KB of fixed arrays)

size_t prefix_smem(int hd, int rows, int psteps, int spages, int group) {
	auto of = [&](auto head) {
		constexpr int HD = decltype(head)::value;
		return rows == 32 ? PrefixSmem<HD, 32>::bytes(psteps, spages, group) : PrefixSmem<HD, 16>::bytes(psteps, spages, group);
	};
	if (hd == 128) return of(std::integral_constant<int, 128>{});
	return hd == 64 ? of(std::integral_constant<int, 64>{}) : of(std::integral_constant<int, 32>{});
}

// tiles of `tq` rows that `rows` rows in `groups` groups need at most
int prefix_tiles(int rows, int groups, int tq) { return std::min<int64_t>(rows, ((int64_t)rows + (int64_t)groups * (tq - 1)) / tq); }

bool prefix_shape(int hd, int rows, int group, int shift, int max_prefix, int max_suffix, PrefixPlan* p) {
	p->rows = rows;
	p->tq = rows / group;
	p->shift = shift;
	const int sub = 1 << shift;
	p->psteps = ((max_prefix + kPfxStep - 1) / kPfxStep + sub - 1) / sub;
	p->spages = (p->tq * ((max_suffix + kPageTokens - 1) / kPageTokens) + sub - 1) / sub;
	p->spages = (p->spages + kPfxStepPages - 1) / kPfxStepPages * kPfxStepPages;
	p->smem = prefix_smem(hd, rows, p->psteps, p->spages, group);
	return p->smem <= kPfxSmemMax;
}

// How a call is cut. False when nothing fits (rows wider than 32,768 positions).
bool prefix_plan(int hd, int group, int kv_heads, int rows, int groups, int max_prefix, int max_suffix, int forced, PrefixPlan* out) {
	const int sms = sm_count();
	bool found = false;
	for (int r : {32, 16}) {
		PrefixPlan best{};
		bool have = false;
		const int top = r == 32 ? 3 : 4;
		for (int shift = 0; shift <= top; ++shift) {
			PrefixPlan p;
			if (!prefix_shape(hd, r, group, shift, max_prefix, max_suffix, &p)) continue;
			p.tiles = prefix_tiles(rows, groups, p.tq);
			if (forced > 0) {
				best = p;
				have = true;
				if (1 << shift >= forced) break;
				continue;
			}
			const int64_t blocks = (int64_t)p.tiles * kv_heads << shift;
			if (have && (blocks > 2 * sms || p.psteps * kPfxStepPages + p.spages < kPfxStepPages)) break;
			best = p;
			have = true;
		}
		if (!have) continue;
		const int64_t blocks = (int64_t)best.tiles * kv_heads << best.shift;
		if (!found || blocks > 0) *out = best;
		found = true;
		if (forced > 0 ? r == 32 : blocks >= sms / 2) break;
	}
	return found;
}

template <int HD, int ROWS, bool RESIDENT>
cudaError_t prefix_launch(const PrefixArgs& a, const PrefixPlan& p, cudaStream_t st) {
	static PerDeviceOnce once;
	const auto kernel = k_attention_prefix<HD, ROWS, RESIDENT>;
	cudaError_t e = once_per_device(once, [&] {
		cudaError_t x = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPfxSmemMax);
		if (x == cudaSuccess) x = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
		if (x == cudaSuccess) x = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
		return x;
	});
	if (e != cudaSuccess) return e;
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3(1u << p.shift, p.tiles, a.kv_heads);
	cfg.blockDim = dim3(kPfxThreads);
	cfg.dynamicSmemBytes = p.smem;
	cfg.stream = st;
	cudaLaunchAttribute attr[2];
	attr[0].id = cudaLaunchAttributeClusterDimension;
	attr[0].val.clusterDim.x = 1u << p.shift;
	attr[0].val.clusterDim.y = 1;
	attr[0].val.clusterDim.z = 1;
	attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[1].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = attr;
	cfg.numAttrs = pdl_enabled() ? 2 : 1;
	return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <bool RESIDENT>
cudaError_t prefix_dispatch(PrefixArgs a, int hd, const PrefixPlan& p, cudaStream_t st) {
	a.tq = p.tq;
	a.ginv = (65536 + a.G - 1) / a.G;
	a.shift = p.shift;
	a.psteps = p.psteps;
	a.spages = p.spages;
	a.debug_withhold = p.shift > 0 ? exchange_debug_take(kExchangeAttnPrefix) : 0;
	if (hd == 128) return p.rows == 32 ? prefix_launch<128, 32, RESIDENT>(a, p, st) : prefix_launch<128, 16, RESIDENT>(a, p, st);
	if (hd == 64) return p.rows == 32 ? prefix_launch<64, 32, RESIDENT>(a, p, st) : prefix_launch<64, 16, RESIDENT>(a, p, st);
	return p.rows == 32 ? prefix_launch<32, 32, RESIDENT>(a, p, st) : prefix_launch<32, 16, RESIDENT>(a, p, st);
}

}  // namespace
}  // namespace sslm

using namespace sslm;

extern "C" sslm_status sslm_b200_attention_prefix_resident(const sslm_b200_prefix_attention* call, void* stream) {
	if (!call || call->struct_size != sizeof(sslm_b200_prefix_attention)) return SSLM_INVALID_ARGUMENT;
	const sslm_b200_prefix_attention& c = *call;
	if (c.rows < 0 || c.groups < 0 || c.reserved != 0) return SSLM_INVALID_ARGUMENT;
	if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) return SSLM_INVALID_ARGUMENT;
	if (c.kv_heads < 1 || c.kv_heads > 65535 || c.heads < 1 || c.heads % c.kv_heads != 0 || c.heads / c.kv_heads > 8) return SSLM_INVALID_ARGUMENT;
	if (c.max_prefix < 0 || c.max_suffix < 0 || c.max_prefix > kPfxMaxWidth || c.max_suffix > kPfxMaxWidth) return SSLM_INVALID_ARGUMENT;
	const int64_t width = (int64_t)c.heads * c.head_dim;
	if (c.num_pages < 0 || c.num_pages > INT32_MAX || c.q_stride < width || c.out_stride < width) return SSLM_INVALID_ARGUMENT;
	const int prefix_pages = (c.max_prefix + kPageTokens - 1) / kPageTokens, suffix_pages = (c.max_suffix + kPageTokens - 1) / kPageTokens;
	if (c.prefix_stride < prefix_pages || c.suffix_stride < suffix_pages) return SSLM_INVALID_ARGUMENT;
	if (c.out_codes && !c.row_status) return SSLM_INVALID_ARGUMENT;
	if (c.rows == 0 || c.groups == 0) return SSLM_OK;
	if (!c.q || !c.consts || !c.group_start || !c.prefix_len || !c.suffix_len || !c.out || (prefix_pages > 0 && !c.prefix_pages) ||
	    (suffix_pages > 0 && !c.suffix_pages) || (!c.kv && c.num_pages > 0) || c.rows > 65535 || c.groups > 65535)
		return SSLM_INVALID_ARGUMENT;
	auto off = [](const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) != 0; };
	if (off(c.kv, 16) || off(c.q, 4) || (c.q_stride & 3) || off(c.out, 16) || (c.out_stride & 3) || off(c.consts, 8) || off(c.out_scales, 8) ||
	    off(c.out_codes, 4) || off(c.group_start, 4) || off(c.prefix_len, 4) || off(c.prefix_pages, 4) || off(c.suffix_len, 4) || off(c.suffix_pages, 4) ||
	    off(c.fold, 4) || off(c.row_status, 4))
		return SSLM_MISALIGNED_BUFFER;
	const int G = c.heads / c.kv_heads;
	PrefixPlan p;
	if (!prefix_plan(c.head_dim, G, c.kv_heads, c.rows, c.groups, c.max_prefix, c.max_suffix, attn_forced_splits(), &p)) return SSLM_INVALID_ARGUMENT;
	PrefixArgs a{};
	a.rows = c.rows; a.groups = c.groups; a.G = G; a.kv_heads = c.kv_heads;
	a.max_prefix = c.max_prefix; a.max_suffix = c.max_suffix;
	a.q = c.q; a.q_stride = c.q_stride;
	a.kv = c.kv; a.num_pages = c.num_pages;
	a.group_start = c.group_start; a.prefix_len = c.prefix_len;
	a.consts = c.consts;
	a.prefix_pages = c.prefix_pages; a.prefix_stride = c.prefix_stride;
	a.suffix_len = c.suffix_len; a.suffix_pages = c.suffix_pages; a.suffix_stride = c.suffix_stride;
	a.fold = c.fold;
	a.out = c.out; a.out_stride = c.out_stride;
	a.status = c.row_status;
	cudaStream_t st = (cudaStream_t)stream;
	if (prefix_dispatch<true>(a, c.head_dim, p, st) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	if (c.out_codes &&
	    launch_pdl(k_prefix_codes, dim3(c.rows), dim3(256), 0, st, (const int32_t*)c.out, c.out_stride, (int)width, c.group_start, c.groups,
	               Scale{c.site_m, c.site_e}, c.out_codes, (Scale*)c.out_scales, c.row_status) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}
