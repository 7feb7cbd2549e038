// Integer i-exp softmax attention of rows that share a prefix, the prefix computed once for all of them.
//
// Rows (one token of one sequence each) come in groups; the rows of a group see the same P positions and
// then S_r of their own. The arithmetic of a row is that of k_attention (sslm_attn.cu), over P + S_r positions:
//   s_k = q . K_k,  e_k = i-exp(s_k - max),  p_k = floor(2^15 e_k / sum),  ctx = sum p_k V_k,  fold
// A tile is ROWS query rows of one kv head: tq = ROWS / G rows of a group times the G q heads of that kv head.
// The tile multiplies the prefix's K and V once, ROWS rows at a time; a row's own pages are multiplied
// with the same instructions, the other rows of the tile left out. A tile is cut over the blocks of a
// cluster, the pages of the prefix and those of the suffixes both dealt round-robin, and the blocks exchange
// maxima, sums and shares of P.V as k_attention_chunk's do (sums and maxima of integers: no order of arrival
// changes a result).
//
// K and V go from L2 straight into the registers of the warp that multiplies them: a page of K belongs to one
// warp, 8 or 16 channels of all V pages to one. The scores stay in shared memory, of the prefix by page and row, of suffix
// pages by page and head, since only G of the tile's rows see such a page; (shift, base) words and then the two
// byte planes of the probabilities take their place. (Both staged through shared memory by double-buffered asynchronous
// copies cost twice the time of the contractions; what room is left takes V pages by bulk copies during the softmax.)
//
// Exactness forbids the running maximum of a floating-point softmax: an element's floors depend on the row's maximum, and its
// probability on the row's sum. So a tile walks its scores three times (maximum; exponentials and sum; probabilities), and holds
// them: 16 or 32 rows x 4 bytes a position, which is what sets the least number of blocks a long prefix takes.
//
// What bounds it (us, one B200, tensors not in L2): one row behind 512 positions of 12 x 128 heads 8.6, eight rows behind 300
// 8.8: the chain (lists and pages 2.5, scores 0.7, three exchanges or barriers 2, softmax 1.5, P.V and store 1.5), bytes under 0.1.
// 64 rows behind 2,048 of 12 x 128 19.6; 256 rows in six ragged groups 35.8, of which the longest tile takes 34 and half of the
// blocks 22; 32 rows behind 16,384 of 16 x 128 66: softmax elements, some 80 instructions each with the contractions, issued in
// 42 % of the slots by sixteen warps, in two rounds, since 192 blocks are needed to hold the scores.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/sslm_b200.h"
#include "sslm_cluster.cuh"
#include "sslm_kernels.h"
#include "sslm_quad.cuh"
#include "sslm_softmax.cuh"

namespace sslm {

constexpr int kPfxThreads = 512;
constexpr int kPfxMaxWidth = 32768;      // positions a row sees at most: the longest admitted context
constexpr int kPfxTokens = 32;           // rows a tile holds at most (32 query rows of groups of one)

struct PrefixArgs {
	int rows, groups, G, kv_heads, tq, ginv, sub;        // ginv = ceil(65536 / G); a tile is cut over `sub` blocks, one cluster
	uint32_t sinv;                                       // ceil(2^32 / sub), of more than one block
	int per, pinv;                                       // rows of the tile that each of them adds up and stores, ceil(65536 / per)
	int ppages, spages;                                  // prefix and suffix pages a block has room for (multiples of four)
	int vgroups;                                         // groups of four pages whose V it has room for
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

// Scores of a page: 64 bytes per row (16 positions), and 16 more, so that the sixteen bytes of four neighbouring
// pages that a lane quad reads together lie in different banks.
constexpr int kPfxPad = 16;
template <int HD, int ROWS>
struct PrefixSmem {
	static constexpr int kQStride = HD + 16, kSumStride = HD + 8;      // (padding against bank conflicts)
	__host__ __device__ static constexpr size_t kShares(int sub) { return (size_t)sub * ((ROWS + sub - 1) / sub) * HD * 4; }      // what the blocks of the cluster send of P.V
	static constexpr size_t kSums = (size_t)ROWS * kSumStride * 4;     // the warps' shares of it, and before that the tile's q rows
	static constexpr size_t bytes(int ppages, int spages, int group, int sub) {
		return (sub > 1 ? kShares(sub) : 0) + kSums + (size_t)ppages * (ROWS * 64 + kPfxPad) + (size_t)spages * (group * 64 + kPfxPad) + (size_t)(ppages + spages) * 12 +
		       (size_t)spages * 4;
	}
	static constexpr size_t kVPage = (size_t)kPageTokens * HD + 32;    // a staged V page (padding as above)
};

// the constants of a row's softmax element lie where the kernels' short forms hold, and a row of `width` such
// elements adds up in 63 bits (the gates of the q/k/v site)
__device__ __forceinline__ bool softmax_gate(int64_t ln2, int64_t qb, int64_t qc, int width) {
	if (ln2 < 1 || ln2 > qb || qb >= (1 << 24) || qc < 0 || qc > SSLM_SOFTMAX_MAX_SAFE) return false;
	const int64_t peak = qb * qb + qc;      // (below 2^49)
	return peak <= SSLM_SOFTMAX_MAX_SAFE && (unsigned long long)peak * (unsigned long long)max(width, 1) <= 0x7FFFFFFFFFFFFFFFull;
}
// The HD / 16 words of a head-dim row that lane column c feeds to the score MMAs: MMA j takes words 2j (k slots 4c ..) and 2j + 1
// (16 + 4c ..), of q and of K alike. A lane's 32 bytes of a row of 128 channels come by one load, which wants them on a 32-byte
// boundary, or (WHOLE false: the pool does not begin on one) by two of 16. A kernel each: with the choice in one, 64 rows behind 2,048 positions took
// 20.0 us in place of 19.8, 256 in six groups 37.5 in place of 37.0, and as much with two loads for all.
template <int HD, bool WHOLE>
__device__ __forceinline__ void row_words(const int8_t* row, int c, uint32_t (&w)[HD / 16]) {
	if constexpr (HD == 128) {
		if constexpr (WHOLE) {
			asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
			             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
			             : "l"(row + c * 32)
			             : "memory");
		} else {
			asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(row + c * 32) : "memory");
			asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(row + c * 32 + 16) : "memory");
		}
	} else if constexpr (HD == 64) {
		asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(row + c * 16) : "memory");
	} else {
		asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(row + c * 8) : "memory");
	}
}
__device__ __forceinline__ int4 load16(const void* p) {
	int4 v;
	asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
	return v;
}

// One softmax element as chunk_exp (sslm_softmax.cuh) has it, under the same gates, with the division by a product: for
// d = q_ln2 <= 2^L, L <= 24, M = floor(2^(31 + L) / d) + 1 fits 32 bits and exceeds 2^(31 + L) / d by at most d / d, so that
// x M / 2^(31 + L) exceeds x / d by at most x / 2^(31 + L) < 1 / d for x <= 30 d, and its floor is that of x / d.
struct IExpMul {
	uint32_t ln2, clip, mul, shift;      // clip = 30 ln2
	int64_t qc;
	uint32_t qb, pad;
};
__device__ __forceinline__ IExpMul iexp_mul_prepare(int64_t ln2, int64_t qb, int64_t qc) {
	IExpMul f;
	f.ln2 = (uint32_t)ln2;
	f.clip = 30u * f.ln2;
	f.shift = 31u + (f.ln2 > 1u ? 32u - (uint32_t)__clz((int)(f.ln2 - 1u)) : 0u);
	// floor(2^shift / d) from a float quotient (off by 2^-22 of 2^32 at most) and two remainders
	const float r = 1.0f / (float)f.ln2;
	const unsigned long long n = 1ull << f.shift;
	uint32_t m = (uint32_t)fminf(r * (float)n, 4294966784.0f);
	m += (uint32_t)(int)floorf((float)(long long)(n - (unsigned long long)m * f.ln2) * r);
	const long long rem = (long long)(n - (unsigned long long)m * f.ln2);
	m += rem >= (long long)f.ln2 ? 1u : 0u;
	m -= rem < 0 ? 1u : 0u;
	f.mul = m + 1u;
	f.qc = qc;
	f.qb = (uint32_t)qb;
	f.pad = 0;
	return f;
}
__device__ __forceinline__ unsigned long long iexp_mul(uint32_t dq, const IExpMul& f, uint32_t* parts) {
	const uint32_t x = min(dq, f.clip);
	const uint32_t z = (uint32_t)(((unsigned long long)x * f.mul) >> f.shift);
	const uint32_t base = z * f.ln2 + (f.qb - x);      // 1 .. q_b < 2^24
	*parts = (z << 24) + base;
	return ((unsigned long long)base * base + (unsigned long long)f.qc) >> z;
}

template <int HD, int ROWS, bool RESIDENT, bool WHOLE>
__global__ void __launch_bounds__(kPfxThreads, 1) k_attention_prefix(const __grid_constant__ PrefixArgs a) {
	using L = PrefixSmem<HD, ROWS>;
	constexpr int KS = HD / 32;                 // MMA steps along the head dimension
	constexpr int RB = ROWS / 16;               // 16-row blocks
	constexpr int W = kPfxThreads / 32;
	constexpr int kPageScores = ROWS * 64 + kPfxPad;
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ __align__(8) unsigned long long s_bars[4];      // staged V; maxima, sums, shares of P.V
	__shared__ unsigned long long s_sum[ROWS], s_rxsum[kPfxThreads];
	__shared__ IExpMul s_fx[kPfxTokens];
	__shared__ float4 s_prob[ROWS];             // (c, q_c, eps) of a row's probabilities
	__shared__ int32_t s_max[ROWS], s_rxmax[kPfxThreads], s_len[kPfxTokens], s_code[kPfxTokens], s_cum[kPfxTokens + 1], s_fold[24], s_tile[4];

	const int G = a.G, kvh = (int)blockIdx.z;
	const int sub = a.sub, rank = (int)blockIdx.x;
	const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, c = lane & 3;
	int32_t* rx_ctx = (int32_t*)smem;                                                       // [sub][per][HD], of a cluster
	int32_t* ctx = (int32_t*)(smem + (sub > 1 ? L::kShares(sub) : 0));                           // [ROWS][kSumStride]
	int8_t* qs = (int8_t*)ctx;                                                              // [ROWS][kQStride]
	unsigned char* vst = (unsigned char*)ctx + L::kSums;                                    // [4 vgroups] staged V pages
	unsigned char* sc = vst + (size_t)a.vgroups * 4 * L::kVPage;                            // [page][row][16] scores of prefix pages
	unsigned char* csc = sc + (size_t)a.ppages * kPageScores;                               // [page][head][16] scores of suffix pages
	const int csc_page = G * 64 + kPfxPad;
	int64_t* pbase = (int64_t*)(csc + (size_t)a.spages * csc_page);                         // page offsets inside a plane, -1: none
	int64_t* sbase = pbase + a.ppages;
	int32_t* sown = (int32_t*)(sbase + a.spages);                                           // owner | positions << 8
	uint32_t* redo = (uint32_t*)(sown + a.spages);                                          // [ppages, then spages] rows whose probabilities need the exact form

	if (t == 0) {
		const int held = (blockIdx.x | blockIdx.y | blockIdx.z) == 0 ? a.debug_withhold : 0;
		ring_init(cta_addr(&s_bars[0]), held == 4 ? 2 : 1);
		if (sub > 1) {
			auto more = [&](int i) { return held == i + 1 ? 4u : 0u; };
			exchange_init(cta_addr(&s_bars[1]), (uint32_t)(sub * ROWS * 4) + more(0));
			exchange_init(cta_addr(&s_bars[2]), (uint32_t)(sub * ROWS * 8) + more(1));
			exchange_init(cta_addr(&s_bars[3]), (uint32_t)(sub * max(0, min(a.per, ROWS - rank * a.per)) * HD * 4) + more(2));
		}
		exchange_fence_init();
	}
	if (sub > 1) {
		__syncwarp();
		cluster_arrive();      // (waited for ahead of the first word that is sent)
	}
	// A caller's tensors may have been written by the kernel in front. Of an engine call the descriptors, lengths and page tables were uploaded, and
	// the prefix's pages filled, before its first launch, but for the ids of pages that the call opens: k_begin enters those. Two kernels lie between
	// (the projections and the q/k/v site), and each waits for the one in front before it lets the next one start, so k_begin is over here.
	if (RESIDENT) {
		pdl_wait();
		pdl_release();
	}
	const int fold_word = t < 3 * G ? (a.fold != nullptr ? a.fold[3 * kvh * G + t] : (t % 3 == 0 ? 1 : 0)) : 0;      // (wanted at the end)
	// ---- which tile: group after group, tq rows at a time
	if (warp == 0) {
		int want = (int)blockIdx.y, r0 = 0, nt = 0, group = 0, prefix = 0;
		if (a.groups == 1) {      // (alike for all lanes)
			const int start = max(a.group_start[0], 0), n = max(min(a.group_start[1], a.rows) - start, 0), len = a.prefix_len[0];
			if (want < (n + a.tq - 1) / a.tq) {
				r0 = start + want * a.tq;
				nt = min(a.tq, n - want * a.tq);
				prefix = len;
			}
		}
		for (int g0 = 0; g0 < a.groups && a.groups > 1; g0 += 32) {
			int start = 0, n = 0, len = 0;
			if (g0 + lane < a.groups) {
				start = a.group_start[g0 + lane];
				n = a.group_start[g0 + lane + 1];
				len = a.prefix_len[g0 + lane];
				start = max(start, 0);
				n = max(min(n, a.rows) - start, 0);
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
				prefix = __shfl_sync(0xffffffffu, len, src);
				group = g0 + src;
				break;
			}
			want -= __shfl_sync(0xffffffffu, upto, 31);
		}
		if (lane == 0) {
			s_tile[0] = r0;
			s_tile[1] = nt;
			s_tile[2] = group;
			s_tile[3] = prefix;
		}
	}
	if (t < ROWS) {
		s_max[t] = INT32_MIN;
		s_sum[t] = 0ull;
	}
	__syncthreads();
	const int r0 = s_tile[0], nt = s_tile[1];
	if (nt == 0) {      // (all blocks of the cluster alike)
		if (sub > 1) cluster_wait();
		return;
	}
	int P = s_tile[3];
	const int32_t* prefix_pages = RESIDENT ? a.prefix_pages + (int64_t)s_tile[2] * a.prefix_stride : a.desc[r0].pages;
	auto stage_q = [&](int first, int step) {      // rows of tokens that there are not: zeros
		constexpr int kWords = ROWS * (HD / 4), kTurns = (kWords + kPfxThreads - 33) / (kPfxThreads - 32);
		uint32_t x[kTurns];
#pragma unroll
		for (int u = 0; u < kTurns; ++u) {      // (all of them on their way before the first is stored)
			const int i = first + u * step, rho = i / (HD / 4), w = i % (HD / 4), tk = rho * a.ginv >> 16;
			x[u] = i < kWords && tk < nt ? *(const uint32_t*)(a.q + (int64_t)(r0 + tk) * a.q_stride + (int64_t)(kvh * G + rho - tk * G) * HD + 4 * w) : 0u;
		}
#pragma unroll
		for (int u = 0; u < kTurns; ++u) {
			const int i = first + u * step;
			if (i < kWords) *(uint32_t*)(qs + i / (HD / 4) * L::kQStride + 4 * (i % (HD / 4))) = x[u];
		}
	};
	const bool bad_len = RESIDENT && (P < 0 || P > a.max_prefix);
	if (bad_len) P = 0;
	// ---- lengths and constants: what is out of range refuses its row; every block of the tile comes to the same verdict
	const int64_t page_bytes = kPageTokens * HD, plane = a.num_pages * page_bytes;
	const int8_t* kplane = a.kv + (int64_t)(2 * kvh) * plane;
	const int8_t* vplane = kplane + plane;
	auto mine = [&](int n) {      // of n things dealt out: rank, rank + sub, ... (n <= 65,536: the product's error is below 1 / sub)
		return n > rank ? (sub > 1 ? (int)__umulhi((uint32_t)(n - rank + sub - 1), a.sinv) : n) : 0;
	};
	auto known = [&](int id) { return !RESIDENT || (uint64_t)(int64_t)id < (uint64_t)a.num_pages; };
	auto stage_v = [&](int at, int64_t base) {      // the page's V into place `at` (filled-up prefix pages first), while there is room
		if (base < 0 || at >= 4 * a.vgroups) return;
		const uint32_t bar = cta_addr(&s_bars[0]);
		asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"((uint32_t)page_bytes) : "memory");
		asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(cta_addr(vst + (size_t)at * L::kVPage)),
		             "l"(vplane + base), "r"((uint32_t)page_bytes), "r"(bar) : "memory");
	};
	const int np = min(mine((P + kPageTokens - 1) / kPageTokens), a.ppages), np4 = (np + 3) & ~3;      // (filled up to groups of four)
	// Page ids of the rows' own pages, all that the tables have room for, are asked for beside the lengths if a thread each is enough.
	// They lie where the sums of other blocks come in, which are sent when this block's maxima are known.
	int32_t* ids = (int32_t*)s_rxsum;
	const int room = (a.max_suffix + kPageTokens - 1) / kPageTokens, own_room = RESIDENT && nt * room <= kPfxThreads - 32 ? room : 0;
	bool bad_page = false;
	if (warp == 0) {
		int code = lane < nt ? kOk : 1, len = 0;
		if (RESIDENT) {
			if (lane < nt) len = a.suffix_len[r0 + lane];
			const int all = nt * a.kv_heads;
			int64_t k[3];
			auto consts_of = [&](int x) {
				const int64_t* from = a.consts + ((int64_t)r0 * a.kv_heads + min(x, all - 1)) * 3;
#pragma unroll
				for (int i = 0; i < 3; ++i) k[i] = from[i];
			};
			consts_of(lane);      // (with the lengths)
			if (lane < nt && (bad_len || len < 0 || len > a.max_suffix || P + len > kPfxMaxWidth)) {
				code = SSLM_B200_ROW_LENGTH;
				len = 0;
			}
			s_code[lane] = 0;
			__syncwarp();
			for (int x0 = 0; x0 < all; x0 += 32) {      // a row's constants of every kv head: a lane each
				const int tk = min((x0 + lane) / a.kv_heads, nt - 1);
				if (x0 > 0) consts_of(x0 + lane);
				if (!softmax_gate(k[0], k[1], k[2], P + __shfl_sync(0xffffffffu, len, tk))) s_code[tk] = SSLM_B200_ROW_CONSTANTS;
			}
			__syncwarp();
			if (code == kOk && s_code[lane] != 0) {
				code = SSLM_B200_ROW_CONSTANTS;
				len = 0;
			}
		} else if (lane < nt) {
			len = min(max(a.desc[r0 + lane].pos + 1 - P, 0), a.max_suffix);
		}
		s_len[lane] = len;
		s_code[lane] = code;
		int upto = (len + kPageTokens - 1) / kPageTokens;      // pages of the suffixes, counted up row by row
#pragma unroll
		for (int o = 1; o < 32; o *= 2) {
			const int v = __shfl_up_sync(0xffffffffu, upto, o);
			if (lane >= o) upto += v;
		}
		s_cum[lane + 1] = upto;
		if (lane == 0) s_cum[0] = 0;
	} else {      // (meanwhile the others: this block's prefix pages, and the tile's q rows)
		for (int i = warp - 1 + lane * (W - 1); i < np4; i += kPfxThreads - 32) {      // (a few of the bulk copies per warp)
			const int id = i < np ? prefix_pages[rank + i * sub] : 0;
			bad_page = bad_page || !known(id);
			pbase[i] = i < np && known(id) ? (int64_t)id * page_bytes : -1;
			redo[i] = 0u;
			stage_v(i, pbase[i]);
		}
		if (RESIDENT) {
			if (t - 32 < nt * own_room) ids[t - 32] = a.suffix_pages[(int64_t)(r0 + (t - 32) / own_room) * a.suffix_stride + (t - 32) % own_room];
			stage_q(t - 32, kPfxThreads - 32);
		}
	}
	// a page id that does not exist: the rows that see the page report the largest maximum there is, which no score
	// reaches, and every block of the tile learns of it with the maxima
	if (__syncthreads_or((int)bad_page) && t < ROWS) s_max[t] = INT32_MAX;
	// ---- K of this warp's first page is on its way while the suffix tables are made
	const int krow = 4 * (g >> 1) + (g & 1);      // position of column g in the first MMA of a page, two more in the second
	uint32_t kn[2][2][HD / 16];      // [page on its way][MMA]
#pragma unroll
	for (int u = 0; u < 2; ++u)
#pragma unroll
		for (int w = 0; w < HD / 16; ++w) kn[u][0][w] = kn[u][1][w] = 0u;
	auto fetch_k = [&](uint32_t (&k)[2][HD / 16], int64_t base) {      // (no page: nothing, the words are not used)
		if (base >= 0) {
			row_words<HD, WHOLE>(kplane + base + krow * HD, c, k[0]);
			row_words<HD, WHOLE>(kplane + base + (krow + 2) * HD, c, k[1]);
		}
	};
#pragma unroll
	for (int u = 0; u < 2; ++u)      // (of an engine call too: the prefix has been in place since its first launch)
		if (warp + u * W < np) fetch_k(kn[u], pbase[warp + u * W]);
	const int ns = min(mine(s_cum[kPfxTokens]), a.spages), ns4 = (ns + 3) & ~3;
	for (int i = warp + lane * W; i < ns4; i += kPfxThreads) {
		int64_t base = -1;
		int own = 255;
		if (i < ns) {
			const int x = rank + i * sub;
			int tk = 0;
			while (s_cum[tk + 1] <= x) ++tk;
			const int page = x - s_cum[tk];
			const int32_t* pages = RESIDENT ? a.suffix_pages + (int64_t)(r0 + tk) * a.suffix_stride : a.desc[r0 + tk].pages + P / kPageTokens;
			const int id = own_room > 0 ? ids[tk * own_room + page] : pages[page];
			if (known(id)) {
				base = (int64_t)id * page_bytes;
				own = tk | min(kPageTokens, s_len[tk] - page * kPageTokens) << 8;
			} else {
				for (int h = 0; h < G; ++h) s_max[tk * G + h] = INT32_MAX;      // (any number of pages may write it)
			}
		}
		sbase[i] = base;
		sown[i] = own;
		redo[a.ppages + i] = 0u;
		if (RESIDENT) stage_v(np4 + i, base);
	}
	if (!RESIDENT) {
		pdl_wait();
		pdl_release();
		stage_q(t, kPfxThreads);
		for (int i = warp + lane * W; i < ns; i += kPfxThreads) stage_v(np4 + i, sbase[i]);      // (the thread's own entries)
		if (t < nt) s_code[t] = __ldcg(&a.status[r0 + t]) != 0 ? 1 : kOk;
		__syncthreads();
	}
	if (warp == W - 1) {      // (wanted by the softmax only)
		IExpConsts k{1, 1, 0};      // (of a row that is left out)
		if (s_code[lane] == kOk) {
			if (RESIDENT) {
				const int64_t* p = a.consts + ((int64_t)(r0 + lane) * a.kv_heads + kvh) * 3;
				k = IExpConsts{p[0], p[1], p[2]};
			} else {
				k = a.smc[(size_t)(r0 + lane) * a.kv_heads + kvh].c;
			}
		}
		s_fx[lane] = iexp_mul_prepare(k.q_ln2, k.q_b, k.q_c);
	}
	if (t < 3 * G) s_fold[t] = fold_word;
	__syncthreads();
	if (t == 0) ring_arrive(cta_addr(&s_bars[0]));      // (every staged page is announced)

	bool ok = true;

	// ---- pass 1: scores and row maxima, a page per warp and turn, K straight into registers. The 16 positions of a page are
	// spread over the columns of two MMAs so that a lane is left with positions 4 c .. 4 c + 3 of its rows.
	{
		uint32_t q[RB][2][HD / 16];
		int tok[RB][2], head[RB][2], mx[RB][2];      // of rows 16 b + 8 e + g
#pragma unroll
		for (int b = 0; b < RB; ++b)
#pragma unroll
			for (int e = 0; e < 2; ++e) {
				const int rho = 16 * b + 8 * e + g;
				tok[b][e] = rho * a.ginv >> 16;
				head[b][e] = rho - tok[b][e] * G;
				mx[b][e] = INT32_MIN;
				const int8_t* row = qs + rho * L::kQStride + c * (HD / 4);
				if constexpr (HD == 32) {
					*(uint2*)q[b][e] = *(const uint2*)row;
				} else {
#pragma unroll
					for (int w = 0; w < HD / 16; w += 4) *(uint4*)&q[b][e][w] = *(const uint4*)(row + 4 * w);
				}
			}
		const int total = np + ns;
		uint32_t kw[2][HD / 16];
#pragma unroll
		for (int u = 0; u < 2; ++u)
			if (warp + u * W >= np && warp + u * W < total) fetch_k(kn[u], sbase[warp + u * W - np]);
#pragma unroll 1
		for (int i = warp; i < total; i += W) {
#pragma unroll
			for (int w = 0; w < HD / 16; ++w) {
				kw[0][w] = kn[0][0][w];
				kw[1][w] = kn[0][1][w];
				kn[0][0][w] = kn[1][0][w];
				kn[0][1][w] = kn[1][1][w];
			}
			if (i + 2 * W < total) fetch_k(kn[1], i + 2 * W < np ? pbase[i + 2 * W] : sbase[i + 2 * W - np]);
			const int own = i < np ? 0 : sown[i - np];
			const int end = i < np ? P - (rank + i * sub) * kPageTokens : own >> 8;      // positions of the page that count
#pragma unroll
			for (int b = 0; b < RB; ++b) {
				int acc[2][4];
#pragma unroll
				for (int h = 0; h < 2; ++h) {
#pragma unroll
					for (int x = 0; x < 4; ++x) acc[h][x] = 0;
#pragma unroll
					for (int j = 0; j < KS; ++j)
						mma_s8s8_full(acc[h], q[b][0][2 * j], q[b][1][2 * j], q[b][0][2 * j + 1], q[b][1][2 * j + 1], kw[h][2 * j], kw[h][2 * j + 1]);
				}
#pragma unroll
				for (int e = 0; e < 2; ++e) {
					int4 v = make_int4(acc[0][2 * e], acc[0][2 * e + 1], acc[1][2 * e], acc[1][2 * e + 1]);
					if (end < kPageTokens) {
						v.x = 4 * c < end ? v.x : INT32_MIN;
						v.y = 4 * c + 1 < end ? v.y : INT32_MIN;
						v.z = 4 * c + 2 < end ? v.z : INT32_MIN;
						v.w = 4 * c + 3 < end ? v.w : INT32_MIN;
					}
					const bool sees = i < np || tok[b][e] == (own & 255);
					unsigned char* at = i < np ? sc + i * kPageScores + (16 * b + 8 * e + g) * 64 : csc + (i - np) * csc_page + head[b][e] * 64;
					if (sees) {
						*(int4*)(at + c * 16) = v;
						mx[b][e] = max(mx[b][e], max(max(v.x, v.y), max(v.z, v.w)));
					}
				}
			}
		}
#pragma unroll
		for (int b = 0; b < RB; ++b)
#pragma unroll
			for (int e = 0; e < 2; ++e) {
				int m = mx[b][e];
				m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
				m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
				if (c == 0) atomicMax(&s_max[16 * b + 8 * e + g], m);
			}
	}
	__syncthreads();
	for (int i = t; i < ROWS * L::kSumStride; i += kPfxThreads) ctx[i] = 0;      // (the q rows are read)
	// (V that is not staged: into L2 during the softmax)
	const int pgroups = np4 >> 2, groups = pgroups + (ns4 >> 2);
	for (int i = 4 * a.vgroups + t; i < 4 * groups; i += kPfxThreads) {
		const int64_t base = i < np4 ? pbase[i] : sbase[i - np4];
		if (base >= 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(vplane + base), "r"((uint32_t)page_bytes) : "memory");
	}
	__syncthreads();
	if (sub > 1) {
		cluster_wait();      // (the peers run)
		if (t < sub * ROWS) exchange_send(&s_rxmax[rank * ROWS + t % ROWS], cta_addr(&s_bars[1]), (uint32_t)(t / ROWS), (uint32_t)s_max[t % ROWS]);
		ok = exchange_wait(cta_addr(&s_bars[1]));
		__syncthreads();      // (all of them are sent)
		if (t < ROWS) {
			int m = INT32_MIN;
			for (int i = 0; i < sub; ++i) m = max(m, s_rxmax[i * ROWS + t]);
			s_max[t] = m;
		}
		__syncthreads();
	}
	if (RESIDENT) {
		if (t < nt && s_code[t] == kOk && s_max[t * G] == INT32_MAX) s_code[t] = SSLM_B200_ROW_INDEX;
		__syncthreads();
		// (the tiles of the first kv head start first: what a later one may have to say about a wait comes after this)
		if (kvh == 0 && rank == 0 && t < nt && a.status != nullptr) a.status[r0 + t] = s_code[t];
	}

	// The softmax passes deal out four positions of one row and page at a time. Of prefix pages a thread keeps to one row, two pages
	// a turn; suffix pages have G rows each.
	constexpr int kTurn = kPfxThreads / (ROWS * 4);      // pages side by side
	const int my_row = (t >> 2) % ROWS, my_page = t / (ROWS * 4);
	const int my_tok = min(my_row * a.ginv >> 16, kPfxTokens - 1);
	const int ntask = ns * G * 4;

	// ---- pass 2: exponentials and row totals; a score's place then holds the element's (shift, base)
	{
		auto four = [](int4* at, uint32_t m, const IExpMul& f, bool whole) {
			const int4 v = *at;
			uint32_t p0, p1, p2, p3;
			unsigned long long e0 = iexp_mul(m - (uint32_t)v.x, f, &p0), e1 = iexp_mul(m - (uint32_t)v.y, f, &p1);
			unsigned long long e2 = iexp_mul(m - (uint32_t)v.z, f, &p2), e3 = iexp_mul(m - (uint32_t)v.w, f, &p3);
			if (!whole) {      // masked positions count for nothing
				if (v.x == INT32_MIN) { e0 = 0; p0 = kBaseOfZero; }
				if (v.y == INT32_MIN) { e1 = 0; p1 = kBaseOfZero; }
				if (v.z == INT32_MIN) { e2 = 0; p2 = kBaseOfZero; }
				if (v.w == INT32_MIN) { e3 = 0; p3 = kBaseOfZero; }
			}
			*at = make_int4((int)p0, (int)p1, (int)p2, (int)p3);
			return (e0 + e1) + (e2 + e3);
		};
		{
			const IExpMul f = s_fx[my_tok];
			const uint32_t m = (uint32_t)s_max[my_row];
			unsigned long long sum = 0ull;
			unsigned char* at = sc + my_row * 64 + c * 16;
#pragma unroll 2
			for (int page = my_page; page < np; page += kTurn)
				sum += four((int4*)(at + page * kPageScores), m, f, (rank + page * sub + 1) * kPageTokens <= P);
			sum += __shfl_xor_sync(0xffffffffu, sum, 1);
			sum += __shfl_xor_sync(0xffffffffu, sum, 2);
			if (c == 0 && sum != 0ull) atomicAdd(&s_sum[my_row], sum);
		}
#pragma unroll 1
		for (int u0 = warp * 32; u0 < ntask; u0 += kPfxThreads) {
			const int u = (u0 + lane) >> 2, page = u * a.ginv >> 16, h = u - page * G;
			const int own = page < ns ? sown[page] : 255;
			unsigned long long sum = 0ull;
			const int rho = (own & 255) * G + h;
			if ((own & 255) < nt) sum = four((int4*)(csc + page * csc_page + h * 64 + c * 16), (uint32_t)s_max[rho], s_fx[own & 255], own >> 8 == kPageTokens);
			sum += __shfl_xor_sync(0xffffffffu, sum, 1);
			sum += __shfl_xor_sync(0xffffffffu, sum, 2);
			if (c == 0 && sum != 0ull) atomicAdd(&s_sum[rho], sum);
		}
	}
	__syncthreads();
	if (sub > 1) {
		if (t < sub * ROWS) exchange_send(&s_rxsum[rank * ROWS + t % ROWS], cta_addr(&s_bars[2]), (uint32_t)(t / ROWS), s_sum[t % ROWS]);
		ok = exchange_wait(cta_addr(&s_bars[2])) && ok;
		__syncthreads();      // (all of them are sent)
	}
	if (t < ROWS) {
		unsigned long long s = sub > 1 ? 0ull : s_sum[t];
		if (sub > 1)
			for (int i = 0; i < sub; ++i) s += s_rxsum[i * ROWS + t];
		s_sum[t] = s;
		const float pc = 32768.0f / (float)(s > 1ull ? s : 1ull);      // (chunk_prob)
		const int tk = t * a.ginv >> 16;
		const bool live = tk < nt && s_code[tk] == kOk;      // (the others' probabilities: far below 1, none of them in doubt)
		s_prob[t] = live ? make_float4(pc, (float)s_fx[tk].qc, pc * 1.01f, 0.0f) : make_float4(8.6736174e-19f, 0.0f, -1.0f, 0.0f);
	}
	__syncthreads();

	// ---- pass 3: probabilities, two planes of bytes: of each page and row (low plane, 16 bytes) and (high plane, 16 bytes), in
	// the place of the page's scores
	{
		// true: the exact form is wanted for one of the row's sixteen positions (its four lanes are of one mind)
		auto four = [&](int4 v, const ChunkProb& p, uint32_t* lo, uint32_t* hi) {
			float near = 1.0f;
			const uint32_t p0 = chunk_prob_of((uint32_t)v.x, p, &near), p1 = chunk_prob_of((uint32_t)v.y, p, &near);
			const uint32_t p2 = chunk_prob_of((uint32_t)v.z, p, &near), p3 = chunk_prob_of((uint32_t)v.w, p, &near);
			*lo = pack_plane(p0, p1, p2, p3, 0);
			*hi = pack_plane(p0, p1, p2, p3, 1);
			return (__ballot_sync(0xffffffffu, near < p.eps) >> (lane & 28) & 15u) != 0u;      // (all lanes have read by now)
		};
		auto put = [&](unsigned char* at, uint32_t lo, uint32_t hi) {
			*(uint32_t*)(at + c * 4) = lo;
			*(uint32_t*)(at + 16 + c * 4) = hi;
		};
		auto constants = [&](int rho) {
			const float4 x = s_prob[rho];
			return ChunkProb{x.x, x.y, x.z};
		};
		{
			const ChunkProb p = constants(my_row);
			unsigned char* row = sc + my_row * 64;
#pragma unroll 1
			for (int page = my_page; page < np; page += 2 * kTurn) {
				const bool two = page + kTurn < np;      // (alike for the row's four lanes)
				unsigned char *at = row + page * kPageScores, *next = two ? at + kTurn * kPageScores : at;
				const int4 v0 = *(const int4*)(at + c * 16), v1 = *(const int4*)(next + c * 16);
				uint32_t lo0, hi0, lo1, hi1;
				const bool redo0 = four(v0, p, &lo0, &hi0), redo1 = four(v1, p, &lo1, &hi1);
				if (!redo0) put(at, lo0, hi0);
				else if (c == 0) atomicOr(&redo[page], 1u << my_row);
				if (two && !redo1) put(next, lo1, hi1);
				else if (two && c == 0) atomicOr(&redo[page + kTurn], 1u << my_row);
			}
		}
#pragma unroll 1
		for (int u0 = warp * 32; u0 < ntask; u0 += kPfxThreads) {
			const int u = (u0 + lane) >> 2, page = u * a.ginv >> 16, h = u - page * G;
			const int tk = page < ns ? sown[page] & 255 : 255;
			const bool there = tk < nt;
			uint32_t lo, hi;
			unsigned char* at = csc + page * csc_page + h * 64;
			const bool again = four(there ? *(const int4*)(at + c * 16) : make_int4(0, 0, 0, 0), there ? constants(tk * G + h) : ChunkProb{8.6736174e-19f, 0.0f, -1.0f}, &lo, &hi);
			if (there && !again) put(at, lo, hi);
			else if (there && c == 0) atomicOr(&redo[a.ppages + page], 1u << h);
		}
		for (int i = t; i < (np4 - np) * ROWS; i += kPfxThreads) {      // (pages that fill up the last group)
			int4* at = (int4*)(sc + (np + i / ROWS) * kPageScores + i % ROWS * 64);
			at[0] = at[1] = make_int4(0, 0, 0, 0);
		}
		// The exact form, apart from the loops above (a call in them costs a third of their time): one row and page at a time.
		__syncthreads();
#pragma unroll 1
		for (int i = warp; i < np + ns; i += W) {
			const bool shared = i < np;
			uint32_t rows = shared ? redo[i] : redo[a.ppages + i - np];
			while (rows != 0u) {
				const int r = __ffs(rows) - 1, tk = shared ? r * a.ginv >> 16 : sown[i - np] & 255, rho = shared ? r : tk * G + r;
				rows &= rows - 1u;
				unsigned char* at = shared ? sc + i * kPageScores + r * 64 : csc + (i - np) * csc_page + r * 64;
				uint4 x = make_uint4(0u, 0u, 0u, 0u);
				if (lane < 4) {
					const int4 v = *(const int4*)(at + c * 16);
					x = chunk_prob_exact((uint32_t)v.x, (uint32_t)v.y, (uint32_t)v.z, (uint32_t)v.w, s_fx[tk].qc, s_sum[rho]);
				}
				__syncwarp();
				if (lane < 4) put(at, pack_plane(x.x, x.y, x.z, x.w, 0), pack_plane(x.x, x.y, x.z, x.w, 1));
			}
		}
	}
	__syncthreads();      // everybody's probabilities are there

	// ---- pass 4: P.V. A warp has 16 channels of 32 rows, or 32 of 16, and every KW-th group of four pages: the planes are read once per
	// so many channels (once per 8, a tile per warp, those reads were the bound; per 32 of 32 rows adding up the warps' shares costs more). Lane column c owns
	// page 4 x + c of a group: its 16-byte row of the V page feeds two MMAs (positions 0..7 and 8..15), the row's planes
	// the A side of both.
	ok = ring_wait(cta_addr(&s_bars[0]), 0) && ok;
	{
		constexpr int NT = 4 / RB, CW = HD / (8 * NT), KW = W / CW;      // 8-channel tiles of a warp; warps along channels and pages
		const int ch0 = (warp % CW) * 8 * NT, part = warp / CW;
		int acc[RB][NT][2][4];      // [row block][8-channel tile][plane]
#pragma unroll
		for (int b = 0; b < RB; ++b)
#pragma unroll
			for (int n = 0; n < NT; ++n)
#pragma unroll
				for (int x = 0; x < 4; ++x) acc[b][n][0][x] = acc[b][n][1][x] = 0;
		int4 vn[NT];
		const unsigned char* vsm = vst + (size_t)c * L::kVPage + (ch0 + g) * kPageTokens;
		auto fetch = [&](int x) {
			if (x < a.vgroups) {
#pragma unroll
				for (int n = 0; n < NT; ++n) vn[n] = *(const int4*)(vsm + (size_t)x * 4 * L::kVPage + n * 8 * kPageTokens);
			} else {
				const int64_t base = x < pgroups ? pbase[4 * x + c] : sbase[4 * (x - pgroups) + c];
#pragma unroll
				for (int n = 0; n < NT; ++n) vn[n] = base >= 0 ? load16(vplane + base + (ch0 + n * 8 + g) * kPageTokens) : make_int4(0, 0, 0, 0);
			}
		};
		auto multiply = [&](int b, int pl, const int4& w0, const int4& w1, const int4 (&v)[NT]) {
#pragma unroll
			for (int n = 0; n < NT; ++n) mma_u8s8_full(acc[b][n][pl], w0.x, w1.x, w0.y, w1.y, v[n].x, v[n].y);
#pragma unroll
			for (int n = 0; n < NT; ++n) mma_u8s8_full(acc[b][n][pl], w0.z, w1.z, w0.w, w1.w, v[n].z, v[n].w);
		};
		if (part < groups) fetch(part);
		int x = part;
#pragma unroll 1
		for (; x < pgroups; x += KW) {      // of the prefix
			int4 v[NT];
#pragma unroll
			for (int n = 0; n < NT; ++n) v[n] = vn[n];
			if (x + KW < groups) fetch(x + KW);
			const unsigned char* at = sc + (4 * x + c) * kPageScores + g * 64;
#pragma unroll
			for (int b = 0; b < RB; ++b)
#pragma unroll
				for (int pl = 0; pl < 2; ++pl)
					multiply(b, pl, *(const int4*)(at + 16 * b * 64 + 16 * pl), *(const int4*)(at + (16 * b + 8) * 64 + 16 * pl), v);
		}
#pragma unroll 1
		for (; x < groups; x += KW) {      // of the suffixes: a page has planes of its owner's G rows, the others' are zero
			int4 v[NT];
#pragma unroll
			for (int n = 0; n < NT; ++n) v[n] = vn[n];
			if (x + KW < groups) fetch(x + KW);
			const int page = 4 * (x - pgroups) + c, first = (sown[page] & 255) * G;
			const unsigned char* at = csc + page * csc_page;
#pragma unroll
			for (int b = 0; b < RB; ++b) {
				int4 w[2][2];      // [row][plane]
#pragma unroll
				for (int e = 0; e < 2; ++e) {
					const uint32_t h = (uint32_t)(16 * b + 8 * e + g - first);
					const bool sees = h < (uint32_t)G;
#pragma unroll
					for (int pl = 0; pl < 2; ++pl) w[e][pl] = sees ? *(const int4*)(at + h * 64 + 16 * pl) : make_int4(0, 0, 0, 0);
				}
				multiply(b, 0, w[0][0], w[1][0], v);
				multiply(b, 1, w[0][1], w[1][1], v);
			}
		}
		if (part < groups) {
#pragma unroll
			for (int b = 0; b < RB; ++b)
#pragma unroll
				for (int n = 0; n < NT; ++n)
#pragma unroll
					for (int x = 0; x < 4; ++x)
						atomicAdd(&ctx[(16 * b + 8 * (x >> 1) + g) * L::kSumStride + ch0 + n * 8 + 2 * c + (x & 1)], acc[b][n][0][x] + 256 * acc[b][n][1][x]);
		}
	}
	__syncthreads();

	// ---- per-head context fold (forward_sites.cpp:1889-1896), store, row maximum for the funnel
	auto store = [&](int rho, int ch, int32_t sum) {      // (a warp's elements lie in one row)
		const int tk = rho * a.ginv >> 16, h = rho - tk * G;
		const bool live = tk < nt && s_code[tk] == kOk;
		const int32_t o = fold(sum, s_fold[3 * h], s_fold[3 * h + 1], s_fold[3 * h + 2]);
		if (live) a.out[(int64_t)(r0 + tk) * a.out_stride + (int64_t)(kvh * G + h) * HD + ch] = o;
		if (!RESIDENT) {
			const uint32_t top = __reduce_max_sync(0xffffffffu, live ? abs_u32(o) : 0u);
			if (lane == 0 && top) atomicMax(&a.rowmax[(size_t)(r0 + tk) * 4 + 3], (unsigned long long)top);
		}
	};
	if (sub == 1) {
		for (int e = t; e < ROWS * HD; e += kPfxThreads) store(e / HD, e % HD, ctx[e / HD * L::kSumStride + e % HD]);
	} else {      // the shares go to the blocks that add them up, `per` rows each
		for (int e = t; e < ROWS * HD / 2; e += kPfxThreads) {
			const int rho = e / (HD / 2), ch = 2 * (e % (HD / 2)), to = rho * a.pinv >> 16;
			exchange_send(&rx_ctx[(rank * a.per + rho - to * a.per) * HD + ch], cta_addr(&s_bars[3]), (uint32_t)to, *(const int2*)&ctx[rho * L::kSumStride + ch]);
		}
		ok = exchange_wait(cta_addr(&s_bars[3])) && ok;
		const int rows = min(a.per, ROWS - rank * a.per);
		for (int e = t; e < rows * HD; e += kPfxThreads) {
			int32_t sum = 0;
			for (int i = 0; i < sub; ++i) sum += rx_ctx[i * a.per * HD + e];
			store(rank * a.per + e / HD, e % HD, sum);
		}
	}
	if (__builtin_expect(!__all_sync(0xffffffffu, ok), 0)) {      // (the warp's lanes speak for the tile's rows)
		if (lane < nt && a.status != nullptr) {
			if (RESIDENT) a.status[r0 + lane] = kInternalWaitTimeout;
			else atomicCAS(&a.status[r0 + lane], 0, pack_status(kInternalWaitTimeout, kSiteCtx, a.layer));
		}
		__syncwarp();
		exchange_leave(cta_addr(&s_bars[0]), sub > 1 ? 4 : 1);
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

constexpr size_t kPfxSmemMax = 216 * 1024;      // (beside 9 KB of fixed arrays)
constexpr int kPfxMaxSub = 16;

size_t prefix_smem(int hd, int rows, int ppages, int spages, int group, int sub) {
	auto of = [&](auto head) {
		constexpr int HD = decltype(head)::value;
		return rows == 32 ? PrefixSmem<HD, 32>::bytes(ppages, spages, group, sub) : PrefixSmem<HD, 16>::bytes(ppages, spages, group, sub);
	};
	if (hd == 128) return of(std::integral_constant<int, 128>{});
	return hd == 64 ? of(std::integral_constant<int, 64>{}) : of(std::integral_constant<int, 32>{});
}

// tiles of `tq` rows that `rows` rows in `groups` groups need at most
int prefix_tiles(int rows, int groups, int tq) { return (int)std::min<int64_t>(rows, ((int64_t)rows + (int64_t)groups * (tq - 1)) / tq); }

bool prefix_shape(int hd, int rows, int group, int tq, int sub, int max_prefix, int max_suffix, PrefixPlan* p) {
	p->rows = rows;
	p->tq = tq;
	p->sub = sub;
	p->ppages = (((max_prefix + kPageTokens - 1) / kPageTokens + sub - 1) / sub + 3) & ~3;
	p->spages = ((p->tq * ((max_suffix + kPageTokens - 1) / kPageTokens) + sub - 1) / sub + 3) & ~3;
	p->smem = prefix_smem(hd, rows, p->ppages, p->spages, group, sub);
	if (p->smem > kPfxSmemMax) return false;
	const size_t vgroup = 4 * ((size_t)kPageTokens * hd + 32);      // (kVPage)
	p->vgroups = (int)std::min<size_t>((p->ppages + p->spages) / 4, (kPfxSmemMax - p->smem) / vgroup);
	p->smem += p->vgroups * vgroup;
	return true;
}

template <int HD, int ROWS, bool RESIDENT>
cudaLaunchConfig_t prefix_config(cudaLaunchAttribute (&attr)[2], int sub, int tiles, int kv_heads, size_t smem, cudaStream_t st) {
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3(sub, tiles, kv_heads);
	cfg.blockDim = dim3(kPfxThreads);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = st;
	attr[0].id = cudaLaunchAttributeClusterDimension;
	attr[0].val.clusterDim.x = (unsigned)sub;
	attr[0].val.clusterDim.y = 1;
	attr[0].val.clusterDim.z = 1;
	attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[1].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = attr;
	cfg.numAttrs = pdl_enabled() ? 2 : 1;
	return cfg;
}
// Once per kernel and device: its attributes, and how many clusters of each size run at once. (Clusters lie inside a GPC, whose
// multiprocessors a size may not divide: of 148, 132 are used by clusters of four or six, 130 by five, 120 by eight, 112 by sixteen.)
struct PrefixKernel {
	PerDeviceOnce once;
	int clusters[kMaxDevices][kPfxMaxSub + 1];
};
template <int HD, int ROWS, bool RESIDENT>
cudaError_t prefix_setup(const int** clusters) {
	static PrefixKernel k;
	const auto kernel = k_attention_prefix<HD, ROWS, RESIDENT, true>;
	const auto set = [](auto f) {
		cudaError_t x = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPfxSmemMax);
		if (x == cudaSuccess) x = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
		if (x == cudaSuccess) x = cudaFuncSetAttribute(f, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
		return x;
	};
	const cudaError_t e = once_per_device(k.once, [&] {
		cudaError_t x = set(kernel);
		if constexpr (RESIDENT && HD == 128) x = x == cudaSuccess ? set(k_attention_prefix<HD, ROWS, true, false>) : x;
		for (int sub = 1; sub <= kPfxMaxSub && x == cudaSuccess; ++sub) {
			cudaLaunchAttribute attr[2];
			const cudaLaunchConfig_t cfg = prefix_config<HD, ROWS, RESIDENT>(attr, sub, 1, 1, kPfxSmemMax, nullptr);
			int n = 0;
			if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {      // (a size the device does not have)
				cudaGetLastError();
				n = 0;
			}
			k.clusters[current_device_ordinal()][sub] = n;
		}
		return x;
	});
	*clusters = k.clusters[current_device_ordinal()];
	return e;
}
template <bool RESIDENT>
cudaError_t prefix_clusters(int hd, int rows, const int** clusters) {
	if (hd == 128) return rows == 32 ? prefix_setup<128, 32, RESIDENT>(clusters) : prefix_setup<128, 16, RESIDENT>(clusters);
	if (hd == 64) return rows == 32 ? prefix_setup<64, 32, RESIDENT>(clusters) : prefix_setup<64, 16, RESIDENT>(clusters);
	return rows == 32 ? prefix_setup<32, 32, RESIDENT>(clusters) : prefix_setup<32, 16, RESIDENT>(clusters);
}

// How a call is cut: the tile height and the blocks per tile whose rounds of blocks end first. A block holds its share of the
// prefix's scores and of every suffix of the tile; where both may be so long that no number of blocks has room for a full tile
// (32,768 each: 16 rows of one head need 330 KB a block), tiles of a half or a quarter of the rows are taken, which always fit. Rows
// are spread over all tiles that the same rounds hold: a block's own pages are fewer then (256 rows of 12 x 128 in six groups: 68
// tiles of four instead of 56 of five, 36.5 -> 34.8 us; 256 rows behind 256: 23.5 -> 20.5).
template <bool RESIDENT>
cudaError_t prefix_plan(int hd, int group, int kv_heads, int rows, int groups, int max_prefix, int max_suffix, int forced, PrefixPlan* out) {
	float least = 0.0f;
	for (int cut = 1; cut <= kPfxMaxSub && least == 0.0f; cut *= 2) for (int r : {32, 16}) {
		const int* clusters = nullptr;
		const cudaError_t e = prefix_clusters<RESIDENT>(hd, r, &clusters);
		if (e != cudaSuccess) return e;
		for (int sub = 1; sub <= kPfxMaxSub; ++sub) {
			PrefixPlan p;
			int tq = std::max(r / group / cut, 1);
			if (clusters[sub] < 1 || !prefix_shape(hd, r, group, tq, sub, max_prefix, max_suffix, &p)) continue;
			const int rounds = (int)(((int64_t)prefix_tiles(rows, groups, tq) * kv_heads + clusters[sub] - 1) / clusters[sub]);
			const int64_t room = (int64_t)rounds * clusters[sub] / kv_heads;      // tiles of the same rounds
			if (rows > groups && room >= groups) tq = std::min<int>(tq, (int)((rows - groups) / (room + 1 - groups)) + 1);      // (the least with so few)
			prefix_shape(hd, r, group, tq, sub, max_prefix, max_suffix, &p);
			p.tiles = prefix_tiles(rows, groups, tq);
			float cost = rounds * (8.0f + (r == 32 ? 0.28f : 0.17f) * p.ppages + 0.2f * p.spages);
			if (forced > 0) cost = (float)(sub < forced ? 1000 + forced - sub : sub - forced);
			if (least == 0.0f || cost + 1.0f < least) {
				least = cost + 1.0f;
				*out = p;
			}
		}
	}
	return least > 0.0f ? cudaSuccess : cudaErrorInvalidConfiguration;
}

template <int HD, int ROWS, bool RESIDENT>
cudaError_t prefix_launch(const PrefixArgs& a, const PrefixPlan& p, cudaStream_t st) {
	cudaLaunchAttribute attr[2];
	const cudaLaunchConfig_t cfg = prefix_config<HD, ROWS, RESIDENT>(attr, p.sub, p.tiles, a.kv_heads, p.smem, st);
	if constexpr (RESIDENT && HD == 128)      // (a caller's pool may begin at any 16-byte boundary)
		if (((uintptr_t)a.kv & 31) != 0) return cudaLaunchKernelEx(&cfg, k_attention_prefix<HD, ROWS, true, false>, a);
	return cudaLaunchKernelEx(&cfg, k_attention_prefix<HD, ROWS, RESIDENT, true>, a);
}

template <bool RESIDENT>
cudaError_t prefix_dispatch(PrefixArgs a, int hd, const PrefixPlan& p, cudaStream_t st) {
	a.tq = p.tq;
	a.ginv = (65536 + a.G - 1) / a.G;
	a.sub = p.sub;
	a.sinv = (uint32_t)(((1ull << 32) + p.sub - 1) / p.sub);
	a.per = (p.rows + p.sub - 1) / p.sub;
	a.pinv = (65536 + a.per - 1) / a.per;
	a.ppages = p.ppages;
	a.spages = p.spages;
	a.vgroups = p.vgroups;
	a.debug_withhold = exchange_debug_take(kExchangeAttnPrefix);
	if (hd == 128) return p.rows == 32 ? prefix_launch<128, 32, RESIDENT>(a, p, st) : prefix_launch<128, 16, RESIDENT>(a, p, st);
	if (hd == 64) return p.rows == 32 ? prefix_launch<64, 32, RESIDENT>(a, p, st) : prefix_launch<64, 16, RESIDENT>(a, p, st);
	return p.rows == 32 ? prefix_launch<32, 32, RESIDENT>(a, p, st) : prefix_launch<32, 16, RESIDENT>(a, p, st);
}

}  // namespace

bool prefix_attention_plan(const Dims& d, int rows, int groups, int max_prefix, int max_suffix, PrefixPlan* out) {
	if (prefix_plan<false>(d.head_dim, d.heads / d.kv_heads, d.kv_heads, rows, groups, max_prefix, max_suffix, attn_forced_splits(), out) != cudaSuccess) {
		cudaGetLastError();
		return false;
	}
	out->groups = groups;
	out->max_suffix = max_suffix;
	return true;
}

cudaError_t launch_attention_prefix(const RowBatch& b, const Dims& d, const LayerDev& layer, int layer_index, KvPoolDev pool, const PrefixPlan& plan,
                                    const int32_t* group_start, const int32_t* prefix_len, cudaStream_t st) {
	PrefixArgs a{};
	a.rows = b.m; a.groups = plan.groups; a.G = d.heads / d.kv_heads; a.kv_heads = d.kv_heads;
	a.max_suffix = plan.max_suffix;
	a.q = b.qrot; a.q_stride = d.hidden;
	a.kv = pool.base + kv_plane_offset(d, pool, layer_index, 0, 0); a.num_pages = pool.num_pages;
	a.group_start = group_start; a.prefix_len = prefix_len;
	a.desc = b.rows; a.smc = b.smc; a.rowmax = b.rowmax; a.layer = b.layer;
	a.fold = layer.f_ctx;
	a.out = b.ctxw; a.out_stride = d.hidden;
	a.status = b.status;
	g_prefix_launches.fetch_add(1, std::memory_order_relaxed);
	return prefix_dispatch<false>(a, d.head_dim, plan, st);
}

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
	if (prefix_plan<true>(c.head_dim, G, c.kv_heads, c.rows, c.groups, c.max_prefix, c.max_suffix, attn_forced_splits(), &p) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
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
