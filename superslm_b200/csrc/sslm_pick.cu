// The greedy pick from logits that penalties, biases and masks have changed.
//
// Per row and token v, in 64-bit integers:
//   x = logit[v];  not allowed: x == INT32_MIN, or the row's mask has bit v clear
//   n = occurrences of v among the row's history ids
//   n > 0:  x = x > 0 ? floor(x 2^15 / theta) : -floor(|x| theta / 2^15)     (both toward zero: a penalty's rounding
//           x -= presence + frequency n                                       never turns it into a reward)
//   x += the sum of the row's biases of v
//   x = clamp(x, -(2^31 - 1), 2^31 - 1), or INT32_MIN where v is not allowed
// and the row's token is the lowest index of the largest x, -2 where nothing is allowed.
//
// One pass over the logits. A row is cut over the blocks of a cluster; a block first marks, for its slice of the
// vocabulary, which tokens the history or the biases name, with counts beside them, and which of the others are
// allowed. The others, nearly all, are streamed past, four at a time, and cost a word of shared memory, a nibble of
// one bitmap and a maximum; where it lies is looked up once, at the end. The named tokens are dear (a division, a
// table) and come last, each to one thread: then their logits are in L2 (asked for ahead of the stream, a thousand
// single words a row cost as much as 20 MB of it; worked on in the stream, nearly every other warp stops for one).
//
// Counts lie in a table of the names (TABLE: 1,536 of few rows and 2,560 of many at most, a thread's ids in registers, whoever enters a token works on it),
// or, for longer lists, by token: an id then costs one atomic that nothing waits for, and the bitmaps and the list of named
// tokens are made from the counts (40 rows of 32,768 ids: 33 us with the bitmaps marked id by id, 18.5 so).
//
// What bounds it (us, one B200, logits not in L2): one row of 151,936 6.9 and 21 rows under a schema 10.6: the chain (record,
// lists, marks, one trip to memory, one exchange). 256 rows 43.5, of which the stream takes 28 at 5.6 TB/s (a kernel that only reads:
// 5.9); the marks in front and the named tokens behind it are not hidden, since one row fills a block and two blocks a
// multiprocessor. 64 rows written out 22.6: 79 MB both ways.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/sslm_b200.h"
#include "sslm_cluster.cuh"
#include "sslm_copies.h"
#include "sslm_kernels.h"

namespace sslm {

constexpr int kPickThreads = 512;
constexpr int kPickPass = 24576;            // tokens whose counts a block holds at a time (a multiple of 32)
constexpr int kPickBits = 262144;           // and tokens whose bits it holds at a time, where the counts lie in a table
constexpr int kPickMaxHistory = 65535;      // (a count is 16 bits)
constexpr int kPickTable = 2560;            // names of a row that the table takes
constexpr int kPickChunk = 1024, kPickStages = 4;      // words of four logits that arrive at once, and places for them

struct PickArgs {
	int rows, vocab, shift, slice;      // a row is cut over 1 << shift blocks of `slice` tokens (a multiple of 32)
	int pass;                           // tokens per pass over a slice (a multiple of 32)
	int hash;                           // places of the table, a power of two, or 0
	int list;                           // counts by token: room for named tokens of a pass, all of it or all that the lists can name
	int sums;                           // 1: there are biases
	int stages;
	// a caller's tensors
	const int32_t* logits;
	int64_t logits_stride;
	const int32_t* params;              // [rows][3] theta (Q15), presence, frequency
	const int32_t *history, *history_len;
	int64_t history_stride;
	int max_history, max_bias;
	const int32_t *bias_tokens, *bias_values, *bias_len;
	int64_t bias_stride;
	const uint8_t* masks;
	int64_t mask_stride;
	const int32_t* mask_page;
	int num_masks;
	int32_t *out_tokens, *out_best, *out_logits;
	int64_t out_stride;
	int32_t* status;
	// rows of an engine call
	const PickRow* desc;
	unsigned long long* best;           // [rows] packed (logit, index) keys
	int debug_withhold;                 // tests only (exchange_debug_take)
};

// What the lists of a row name is kept in one of two ways. In a table (TABLE) of places found by the token's hash, with the
// count and the sum of the biases beside each: its size goes by the lists, so a block may have a slice of any length, and a
// thread keeps its ids of the lists in registers from the start of the call. Or, for long lists, as counts of 16 bits by
// token, a list of those that are named, and a table for the biases alone.
struct PickSmem {
	// logits on their way [stages][kPickChunk], sums [hash] if there are biases, tokens [hash], TABLE: counts [hash], else counts u16
	// [pass + 8], bits of the tokens that are allowed and not named, bits of the named ones if kept, else list u16 [list]
	__host__ __device__ static int words(int pass) { return (pass / 32 + 11) & ~3; }      // of a bitmap: filled four at a time (16-byte stores), read one further
	static size_t bytes(bool table, bool out, int stages, int sums, int pass, int hash, int list) {
		return (size_t)stages * kPickChunk * 16 + (size_t)hash * ((table ? 8 : 4) + 8 * sums) + (table ? 0 : (size_t)(pass + 8) * 2) +
		       (size_t)words(pass) * (table && !out ? 4 : 8) + (table ? 0 : (size_t)list * 2);
	}
};

__device__ __forceinline__ unsigned long long pick_key(int32_t x, int v) {
	return x == INT32_MIN ? 0ull : (unsigned long long)((uint32_t)x ^ 0x80000000u) << 32 | (0xFFFFFFFFu - (uint32_t)v);
}

template <bool RESIDENT, bool TABLE, bool OUT>
__global__ void __launch_bounds__(kPickThreads, 2) k_pick(const __grid_constant__ PickArgs a) {
	constexpr bool NAMED = OUT || !TABLE;      // the named bits are kept
	constexpr int kStride = 4 * kPickThreads;
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ __align__(8) unsigned long long s_bar, s_full[kPickStages], s_rx[16], s_warp[kPickThreads / 32];
	__shared__ PickRow s_row;
	__shared__ int s_listed, s_code, s_late, s_part[kPickThreads / 32];
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.vocab;
	const int sub = 1 << a.shift, rank = (int)blockIdx.x;
	const int64_t r = blockIdx.y;
	const int4* ring = (const int4*)smem;                                   // [stages][kPickChunk]
	unsigned long long* bsum = (unsigned long long*)(smem + (size_t)a.stages * kPickChunk * 16);      // [hash], if there are biases
	int32_t* bkey = (int32_t*)(bsum + (a.sums ? a.hash : 0));               // [hash] token, -1: free
	uint32_t* counts = (uint32_t*)(bkey + a.hash);                          // TABLE: [hash], else u16 pairs by token
	uint32_t* dense = counts + (TABLE ? a.hash : (a.pass + 8) / 2);         // bit i: token v0 + i is allowed and not named
	uint32_t* named = dense + (NAMED ? PickSmem::words(a.pass) : 0);
	uint16_t* list = (uint16_t*)(named + PickSmem::words(a.pass));
	const int held = (blockIdx.x | blockIdx.y) == 0 ? a.debug_withhold : 0;
	if (t == 0) {
		if (sub > 1 && rank == 0) exchange_init(cta_addr(&s_bar), (uint32_t)(sub * 8) + (held == 1 ? 4u : 0u));
		for (int i = 0; i < kPickStages; ++i) ring_init(cta_addr(&s_full[i]), 1);
		exchange_fence_init();
		s_late = 0;
	}
	if (sub > 1) {
		__syncwarp();
		cluster_arrive();      // (waited for ahead of the word that is sent)
	}
	pdl_wait();
	pdl_release();

	// ---- the row
	const int32_t* logits = RESIDENT ? a.logits + r * a.logits_stride : a.desc[r].logits;
	int32_t* out = nullptr;
	if (OUT) out = a.out_logits + r * a.out_stride;
	if (t == 0) {
		PickRow x{};
		int32_t code = 0;
		if (RESIDENT) {
			x.theta = 32768;
			x.extra = -1;
			const int page = a.mask_page != nullptr ? a.mask_page[r] : -1;
			if (a.params != nullptr) {
				x.theta = a.params[3 * r];
				x.presence = a.params[3 * r + 1];
				x.frequency = a.params[3 * r + 2];
			}
			if (a.history != nullptr) {
				x.history = a.history + r * a.history_stride;
				x.n_history = a.history_len[r];
			}
			if (a.bias_tokens != nullptr) {
				x.bias_tokens = a.bias_tokens + r * a.bias_stride;
				x.bias_values = a.bias_values + r * a.bias_stride;
				x.n_bias = a.bias_len[r];
			}
			if (page >= 0 && page < a.num_masks) x.mask = a.masks + (int64_t)page * a.mask_stride;
			if (x.theta < 1) code = SSLM_B200_ROW_CONSTANTS;
			if (x.n_history < 0 || x.n_history > a.max_history || x.n_bias < 0 || x.n_bias > a.max_bias) code = SSLM_B200_ROW_LENGTH;
			if (page >= a.num_masks || (page < -1 && code == 0)) code = SSLM_B200_ROW_INDEX;      // (-1, and nothing else below zero, says: no mask)
			if (rank == 0 && a.status != nullptr) a.status[r] = code;
		} else {
			x = a.desc[r];
			if (x.logits == nullptr) code = 1;      // (a row without controls)
			else if (x.extra >= 0 && rank == 0) const_cast<int32_t*>(x.history)[x.n_history] = x.extra;      // (its blocks count it from the record)
		}
		s_row = x;
		s_code = code;
	}
	// TABLE: this thread's ids, asked for with the row's record (of the lists' whole room: how much of it counts is known later)
	constexpr int IH = TABLE ? kPickTable / kPickThreads : 0, IB = TABLE ? kPickMaxBias / kPickThreads : 0, IN = IH + IB + 1;
	int32_t id[IN], add[IB + 1];
	if constexpr (TABLE && RESIDENT) {
#pragma unroll
		for (int u = 0; u < IH; ++u) id[u] = a.history != nullptr && t + u * kPickThreads < a.max_history ? a.history[r * a.history_stride + t + u * kPickThreads] : -1;
#pragma unroll
		for (int u = 0; u < IB; ++u) {
			const bool there = a.bias_tokens != nullptr && t + u * kPickThreads < a.max_bias;
			id[IH + u] = there ? a.bias_tokens[r * a.bias_stride + t + u * kPickThreads] : -1;
			add[u] = there ? a.bias_values[r * a.bias_stride + t + u * kPickThreads] : 0;
		}
	}
	const PickRow& w = s_row;      // (in shared memory: the registers are wanted elsewhere)
	const int s0 = min(V, rank * a.slice), s1 = min(V, s0 + a.slice);
	// four neighbouring tokens of the row lie in one aligned 16-byte word; mis: tokens by which the row's first is off
	const int mis = (int)(((uintptr_t)logits >> 2) & 3), mis_out = (int)(((uintptr_t)out >> 2) & 3);
	int v0 = s0, v1, first, last, chunks;
	uint32_t seq = 0;      // chunks of earlier passes
	CopyAccount copies{(uint32_t)a.stages, 0u};      // (kept by the first thread, which asks for all but a pass's first copies)
	// a pass: tokens v0 .. v1; whole aligned words of four tokens lie from `first` to `last`, the ends are taken one by one
	auto issue = [&](int chunk) {      // (one thread; the place is free)
		const uint32_t at = copies.place(seq + (uint32_t)chunk), bar = cta_addr(&s_full[at]);
		const uint32_t bytes = (uint32_t)min(4 * kPickChunk, last - first - 4 * kPickChunk * chunk) * 4u;
		asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes + (held == 2 && seq + chunk == 0 ? 16u : 0u)) : "memory");
		asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(cta_addr(ring + at * kPickChunk)),
		             "l"(logits + first + 4 * kPickChunk * chunk), "r"(bytes), "r"(bar) : "memory");
	};
	auto begin = [&]() {
		v1 = min(s1, v0 + a.pass);
		first = min(v1, v0 + ((4 - ((v0 + mis) & 3)) & 3));
		last = first + ((v1 - first) & ~3);
		chunks = ((last - first) / 4 + kPickChunk - 1) / kPickChunk;
		if ((uint32_t)t < copies.begin(seq, (uint32_t)chunks)) issue(t);      // (the first of them on their way while the marks are made; one thread for all took 0.5 us longer)
	};
	__syncthreads();
	if (s_code != 0) {      // (all blocks of the cluster alike)
		if (sub > 1) cluster_wait();
		return;
	}
	if (v0 < s1) begin();
	const bool listed = w.n_history > 0 || w.extra >= 0 || w.n_bias > 0;
	if constexpr (TABLE) {
#pragma unroll
		for (int u = 0; u < IH; ++u) {
			if (!RESIDENT) id[u] = t + u * kPickThreads < w.n_history ? w.history[t + u * kPickThreads] : -1;
			else if (t + u * kPickThreads >= w.n_history) id[u] = -1;
		}
#pragma unroll
		for (int u = 0; u < IB; ++u) {
			const bool there = t + u * kPickThreads < w.n_bias;
			if (!RESIDENT) add[u] = there ? w.bias_values[t + u * kPickThreads] : 0;
			id[IH + u] = there ? (RESIDENT ? id[IH + u] : w.bias_tokens[t + u * kPickThreads]) : -1;
		}
		id[IN - 1] = !RESIDENT && t == 0 ? w.extra : -1;
	}
	auto place = [&](int v) { return ((uint32_t)v * 2654435761u) >> 7 & (uint32_t)(a.hash - 1); };
	unsigned long long key = 0ull;
	while (v0 < s1 && s_late == 0) {      // (alike for all: it changes behind a pass's barriers only)
		const int n = v1 - v0, words = (n + 31) / 32;
		// ---- marks and counts of tokens v0 .. v1
		for (int i = 4 * t; i < words + 2; i += 4 * kPickThreads) {
			uint32_t bits[4];
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				const int left = n - (i + j) * 32;
				bits[j] = left >= 32 ? 0xFFFFFFFFu : (left > 0 ? (1u << left) - 1u : 0u);
				if (w.mask != nullptr && left > 0) {      // (v0 is a multiple of 32; a page has ceil(V / 8) bytes and any address)
					const uint8_t* m = w.mask + (v0 >> 3) + 4 * (i + j);
					uint32_t page = 0;
					if (left >= 32 && ((uintptr_t)m & 3) == 0) page = *(const uint32_t*)m;
					else
						for (int b = 0; b < min(4, (left + 7) >> 3); ++b) page |= (uint32_t)m[b] << (8 * b);
					bits[j] &= page;
				}
			}
			*(uint4*)(dense + i) = make_uint4(bits[0], bits[1], bits[2], bits[3]);
			if constexpr (NAMED) *(uint4*)(named + i) = make_uint4(0u, 0u, 0u, 0u);
		}
		int at[IN];      // TABLE: the place of an id that this thread was the first to enter, or -1
#pragma unroll
		for (int u = 0; u < IN; ++u) at[u] = -1;
		if (listed) {
			if constexpr (!TABLE)
				for (int i = t; i < (n + 8) / 8; i += kPickThreads) ((int4*)counts)[i] = make_int4(0, 0, 0, 0);
			for (int i = t; i < a.hash; i += kPickThreads) {
				bkey[i] = -1;
				if (a.sums) bsum[i] = 0ull;
				if constexpr (TABLE) counts[i] = 0u;
			}
			__syncthreads();
			// (a token that is not allowed is the stream's, whoever names it)
			auto enter = [&](int v, bool* new_to_it) {      // its place in the table (a quarter of the places at least stay free)
				uint32_t h = place(v);
				for (;;) {
					int was = *(volatile int32_t*)&bkey[h];
					if (was == -1) {
						was = atomicCAS(&bkey[h], -1, v);
						*new_to_it = was == -1;
						if (was == -1) break;
					}
					if (was == v) break;
					h = (h + 1) & (uint32_t)(a.hash - 1);
				}
				return h;
			};
			if constexpr (TABLE) {
#pragma unroll
				for (int u = 0; u < IN; ++u) {
					const uint32_t i = (uint32_t)(id[u] - v0);
					if (i >= (uint32_t)n) continue;
					bool new_to_it = false;
					const uint32_t h = enter(id[u], &new_to_it);
					if (new_to_it && (atomicAnd(&dense[i >> 5], ~(1u << (i & 31))) >> (i & 31) & 1u) != 0u) {
						at[u] = (int)h;
						if constexpr (NAMED) atomicOr(&named[i >> 5], 1u << (i & 31));
					}
					if (u < IH || u == IN - 1) atomicAdd(&counts[h], 1u);
					else atomicAdd(&bsum[h], (unsigned long long)(long long)add[u - IH]);
				}
			} else {
				auto seen = [&](int v) {
					const uint32_t i = (uint32_t)(v - v0);
					if (i < (uint32_t)n) atomicAdd(&counts[i >> 1], 1u << (16 * (i & 1)));      // (nothing waits for it)
				};
				// (ids of any alignment: single ones up to the first 16-byte word, then words, the next ones asked for ahead)
				const int head = min(w.n_history, (int)((4 - (((uintptr_t)w.history >> 2) & 3)) & 3)), whole = (w.n_history - head) >> 2;
				const int4* ids = (const int4*)(w.history + head);
				auto fetch = [&](int4 (&x)[4], int i0) {
#pragma unroll
					for (int u = 0; u < 4; ++u) x[u] = i0 + u * kPickThreads < whole ? ids[i0 + u * kPickThreads] : make_int4(-1, -1, -1, -1);
				};
				int4 x[4], y[4];
				fetch(x, t);
				for (int i = t; i < w.n_bias; i += kPickThreads) {
					const int v = w.bias_tokens[i];
					const uint32_t at_bit = (uint32_t)(v - v0);
					if (at_bit >= (uint32_t)n) continue;
					bool new_to_it = false;
					atomicAdd(&bsum[enter(v, &new_to_it)], (unsigned long long)(long long)w.bias_values[i]);
					if (new_to_it) atomicOr(&named[at_bit >> 5], 1u << (at_bit & 31));
				}
				if (t < head) seen(w.history[t]);
				for (int i0 = t; i0 < whole; i0 += 4 * kPickThreads) {
					fetch(y, i0 + 4 * kPickThreads);
#pragma unroll
					for (int u = 0; u < 4; ++u) {
						seen(x[u].x);
						seen(x[u].y);
						seen(x[u].z);
						seen(x[u].w);
						x[u] = y[u];
					}
				}
				const int tail = head + 4 * whole + t;
				if (tail < w.n_history) seen(w.history[tail]);
				if (t == 0 && w.extra >= 0) seen(w.extra);
				__syncthreads();
				// a thread's words of the bitmaps, from the counts; the list is of tokens that are counted and have no bias
				constexpr int kWords = (kPickPass / 32 + kPickThreads - 1) / kPickThreads;
				uint32_t counted[kWords];
				int have = 0;
#pragma unroll
				for (int u = 0; u < kWords; ++u) {
					const int i = t + u * kPickThreads;
					counted[u] = 0u;
					if (i >= words) continue;
#pragma unroll
					for (int j = 0; j < 4; ++j) {      // (behind the last token lies something else, which does not count)
						const uint4 q = ((const uint4*)counts)[4 * i + j];
						const uint32_t pair[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
						for (int k = 0; k < 4; ++k)
							counted[u] |= ((pair[k] & 0xFFFFu) != 0u ? 1u << (8 * j + 2 * k) : 0u) | (pair[k] >> 16 != 0u ? 2u << (8 * j + 2 * k) : 0u);
					}
					if (n - 32 * i < 32) counted[u] &= (1u << (n - 32 * i)) - 1u;
					const uint32_t allowed = dense[i], biased = named[i] & allowed;
					counted[u] &= allowed & ~biased;
					named[i] = biased | counted[u];
					dense[i] = allowed & ~(biased | counted[u]);
					have += __popc(counted[u]);
				}
				int upto = have;
#pragma unroll
				for (int o = 1; o < 32; o *= 2) {
					const int z = __shfl_up_sync(0xffffffffu, upto, o);
					if (lane >= o) upto += z;
				}
				if (lane == 31) s_part[warp] = upto;
				__syncthreads();
				int to = upto - have;
				for (int i = 0; i < warp; ++i) to += s_part[i];
				if (t == kPickThreads - 1) s_listed = to + have;
#pragma unroll
				for (int u = 0; u < kWords; ++u)
					for (uint32_t bits = counted[u]; bits != 0u; bits &= bits - 1u) list[to++] = (uint16_t)(32 * (t + u * kPickThreads) + __ffs(bits) - 1);
			}
		}
		__syncthreads();
		// ---- the tokens that nothing names
		auto single = [&](int v) {
			const int i = v - v0;
			const bool use = (dense[i >> 5] >> (i & 31) & 1u) != 0u;
			const int32_t y = use ? logits[v] : INT32_MIN;
			key = max(key, pick_key(y, v));
			if constexpr (OUT) {
				if ((named[i >> 5] >> (i & 31) & 1u) == 0u) out[v] = y;
			}
		};
		if (t < first - v0) single(v0 + t);
		if (t < v1 - last) single(last + t);
		// a thread has every 512th word: their bits lie at one place of their bitmap words
		const int bit = (first - v0 + 4 * t) & 31, word = (first - v0 + 4 * t) >> 5;
		const bool straddles = bit > 28;
		auto nibble = [&](const uint32_t* map, int k) {
			const uint32_t* p = map + word + k * (kStride / 32);
			return __funnelshift_r(p[0], straddles ? p[1] : 0u, bit) & 15u;
		};
		auto words_of = [&](int4 q, uint32_t use, int32_t (&y)[4]) {
			y[0] = q.x; y[1] = q.y; y[2] = q.z; y[3] = q.w;
			if (use != 15u) {
#pragma unroll
				for (int j = 0; j < 4; ++j) y[j] = (use >> j & 1u) != 0u ? y[j] : INT32_MIN;
			}
		};
		int32_t top = INT32_MIN;
		int top_at = 0;      // the word that has it first, and where in it
		const int total = (last - first) / 4;
#pragma unroll 1
		for (int i = 0; i < chunks; ++i) {
			const uint32_t slot = copies.place(seq + (uint32_t)i);
			if (s_late == 0 && !ring_wait(cta_addr(&s_full[slot]), copies.parity(seq + (uint32_t)i))) s_late = 1;      // (what is read then does not count)
#pragma unroll
			for (int u = 0; u < kPickChunk / kPickThreads; ++u) {
				const int k = i * (kPickChunk / kPickThreads) + u;
				if (k * kPickThreads + t >= total) break;
				int32_t y[4];
				words_of(ring[slot * kPickChunk + u * kPickThreads + t], nibble(dense, k), y);
				const int32_t m = max(max(y[0], y[1]), max(y[2], y[3]));
				if (m > top) {
					top = m;
					top_at = 4 * k + (y[0] == m ? 0 : (y[1] == m ? 1 : (y[2] == m ? 2 : 3)));
				}
				if constexpr (OUT) {
					const uint32_t nm = listed ? nibble(named, k) : 0u;
					int32_t* to = out + first + 4 * t + k * kStride;
					if (mis_out == mis && nm == 0u) {
						__stcs((int4*)to, make_int4(y[0], y[1], y[2], y[3]));
					} else {
#pragma unroll
						for (int j = 0; j < 4; ++j)
							if ((nm >> j & 1u) == 0u) to[j] = y[j];
					}
				}
			}
			__syncthreads();      // the place is free
			if (t == 0 && copies.follows((uint32_t)i, (uint32_t)chunks, s_late != 0)) issue(i + a.stages);
		}
		if (top != INT32_MIN) key = max(key, pick_key(top, first + 4 * t + (top_at >> 2) * kStride + (top_at & 3)));
		// ---- the named tokens: (in place, they read as they were)
		if (listed) {
			const double inv_theta = 1.0 / (double)w.theta;
			auto change = [&](int v, int32_t y, uint32_t cnt, long long sum) {      // its logit, its occurrences, what the biases add
				if (y != INT32_MIN) {
					long long z = y;
					if (cnt != 0u) {
						if (z > 0) {      // floor(2^15 z / theta): a quotient in doubles, off by one at most, settled by its remainder
							const long long num = z << 15;
							const long long q = (long long)((double)num * inv_theta), rem = num - q * (long long)w.theta;
							z = q + (rem >= (long long)w.theta ? 1 : 0) - (rem < 0 ? 1 : 0);
						} else {
							z = -((-z * (long long)w.theta) >> 15);
						}
						z -= (long long)w.presence + (long long)w.frequency * (long long)cnt;
					}
					y = (int32_t)max(-2147483647ll, min(2147483647ll, z + sum));
				}
				key = max(key, pick_key(y, v));
				if constexpr (OUT) out[v] = y;
			};
			if constexpr (TABLE) {
				int32_t raw[IN];
#pragma unroll
				for (int u = 0; u < IN; ++u) raw[u] = at[u] >= 0 ? logits[id[u]] : INT32_MIN;
#pragma unroll
				for (int u = 0; u < IN; ++u)
					if (at[u] >= 0) change(id[u], raw[u], counts[at[u]], a.sums ? (long long)bsum[at[u]] : 0ll);
			} else {
				for (int h = t; h < a.hash; h += kPickThreads) {
					const int v = bkey[h];
					if (v >= 0 && (named[(v - v0) >> 5] >> ((v - v0) & 31) & 1u) != 0u) change(v, logits[v], counts[(v - v0) >> 1] >> (16 * ((v - v0) & 1)) & 0xFFFFu, (long long)bsum[h]);
				}
				int32_t y[4];      // (logits of the next four turns)
#pragma unroll
				for (int u = 0; u < 4; ++u) y[u] = t + u * kPickThreads < s_listed ? logits[v0 + list[t + u * kPickThreads]] : INT32_MIN;
#pragma unroll 1
				for (int k = t; k < s_listed; k += kPickThreads) {
					const int i = list[k], ahead = k + 4 * kPickThreads;
					const int32_t x = y[0];
					y[0] = y[1];
					y[1] = y[2];
					y[2] = y[3];
					y[3] = ahead < s_listed ? logits[v0 + list[ahead]] : INT32_MIN;
					change(v0 + i, x, counts[i >> 1] >> (16 * (i & 1)) & 0xFFFFu, 0);
				}
			}
		}
		__syncthreads();      // the tables may be overwritten
		seq += (uint32_t)chunks;
		v0 += a.pass;
		if (v0 < s1 && s_late == 0) begin();
	}
	// ---- the row's largest key: larger values first, then lower indices
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
	if (lane == 0) s_warp[warp] = key;
	if (t == 0 && s_late != 0)      // (a copy that is late may still come, into memory that the next block owns: every place's last one is waited for)
		for (uint32_t i = copies.open(); i < copies.issued; ++i) ring_wait(cta_addr(&s_full[copies.place(i)]), copies.parity(i));
	__syncthreads();
	if (warp != 0) {
		if (sub > 1) cluster_wait();
		return;
	}
	key = lane < kPickThreads / 32 ? s_warp[lane] : 0ull;
#pragma unroll
	for (int o = 8; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
	bool ok = s_late == 0;
	if (sub > 1) {
		cluster_wait();      // (the first block runs)
		if (!ok) key = 1ull;      // (no token's key: theirs have an index below 2^30)
		if (lane == 0) exchange_send(&s_rx[rank], cta_addr(&s_bar), 0u, key);
		if (rank != 0) return;      // (nothing is sent to it)
		ok = exchange_wait(cta_addr(&s_bar)) && ok;
		key = lane < sub ? s_rx[lane] : 0ull;
		ok = !__any_sync(0xffffffffu, key == 1ull) && ok;
#pragma unroll
		for (int o = 8; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
	}
	if (lane == 0 && ok) {
		if (RESIDENT) {
			if (a.out_tokens != nullptr) a.out_tokens[r] = key == 0ull ? -2 : (int32_t)(0xFFFFFFFFu - (uint32_t)key);
			if (a.out_best != nullptr) a.out_best[r] = key == 0ull ? INT32_MIN : (int32_t)((uint32_t)(key >> 32) ^ 0x80000000u);
		} else {
			a.best[r] = key;
		}
	}
	if (__builtin_expect(!__all_sync(0xffffffffu, ok), 0)) {
		if (lane == 0 && a.status != nullptr) {
			if (RESIDENT) a.status[r] = kInternalWaitTimeout;
			else atomicCAS(&a.status[r], 0, pack_status(kInternalWaitTimeout, kSiteLogits, a.desc[r].layer));
		}
		__syncwarp();
		if (sub > 1) exchange_leave(cta_addr(&s_bar), 1);      // (a block by itself has no exchange: its barrier was never set up)
	}
}

namespace {

// names: how many tokens the lists of a row can name; biases of them. True: the table.
bool pick_plan(int names, int biases, PickArgs* a) {
	// The table or counts by token, us: 151,936 tokens and one row 12.3 / 12.3 with 1,600 names and 14.3 / 12.3 with 2,400, 21 rows
	// 16.4 / 18.4 and 20.4 / 18.4 (2,560), but 64 rows 24.6 / 32.8 and 256 rows 74 / 102 (2,560): there the passes that the counts
	// need cost more than a table's turns. 32,003 tokens: one and 21 rows 14.3 / 12.3 (2,400), 64 16.4 / 16.4, 256 31 / 33.
	const bool table = names <= (a->rows <= 32 ? 1536 : kPickTable);
	// blocks per row: as many as run at once, two a multiprocessor, with slices of at least 4,096 tokens; without the table
	// the passes of a slice repeat the lists, so one pass if possible
	const int most = std::max(1, 2 * sm_count() / a->rows);
	a->shift = 0;
	while (a->shift < 4 && a->vocab >> (a->shift + 1) >= 4096 && (2 << a->shift <= most || (!table && a->vocab >> a->shift > kPickPass))) ++a->shift;
	a->slice = (((a->vocab + (1 << a->shift) - 1) >> a->shift) + 31) & ~31;
	a->pass = std::min(a->slice, table ? kPickBits : kPickPass);
	a->list = std::min(a->pass, names);
	a->sums = biases > 0 ? 1 : 0;
	a->hash = 0;
	const int kept = table ? names : biases;
	if (kept > 0) {
		a->hash = 64;
		while (3 * a->hash < 4 * kept) a->hash *= 2;
	}
	// logits on their way: what a pass has, four chunks at most, two where that lets two blocks share a multiprocessor
	const size_t half = 112 * 1024, kept_bytes = PickSmem::bytes(table, a->out_logits != nullptr, 0, a->sums, a->pass, a->hash, a->list), chunk = kPickChunk * 16;
	a->stages = std::max(1, std::min(kPickStages, (a->pass / 4 + kPickChunk - 1) / kPickChunk));
	while (a->stages > 2 && kept_bytes + a->stages * chunk > half && kept_bytes + 2 * chunk <= half) --a->stages;
	return table;
}

template <bool RESIDENT, bool TABLE, bool OUT>
cudaError_t pick_launch(PickArgs a, cudaStream_t st) {
	static PerDeviceOnce once;
	const auto kernel = k_pick<RESIDENT, TABLE, OUT>;
	cudaError_t e = once_per_device(once, [&] {
		const size_t most = TABLE ? PickSmem::bytes(true, true, kPickStages, 1, kPickBits, 4096, 0) : PickSmem::bytes(false, true, kPickStages, 1, kPickPass, 2 * kPickMaxBias, kPickPass);
		const cudaError_t x = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
		return x != cudaSuccess ? x : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
	});
	if (e != cudaSuccess) return e;
	a.debug_withhold = exchange_debug_take(kExchangePick);
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3(1u << a.shift, a.rows);
	cfg.blockDim = dim3(kPickThreads);
	cfg.dynamicSmemBytes = PickSmem::bytes(TABLE, OUT, a.stages, a.sums, a.pass, a.hash, a.list);
	cfg.stream = st;
	cudaLaunchAttribute attr[2];
	attr[0].id = cudaLaunchAttributeClusterDimension;
	attr[0].val.clusterDim.x = 1u << a.shift;
	attr[0].val.clusterDim.y = 1;
	attr[0].val.clusterDim.z = 1;
	attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[1].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = attr;
	cfg.numAttrs = pdl_enabled() ? 2 : 1;
	return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

cudaError_t launch_pick(const PickRow* rows, int m, int vocab, int names, int biases, unsigned long long* best, int32_t* out, int32_t* status, cudaStream_t st) {
	PickArgs a{};
	a.rows = m; a.vocab = vocab;
	a.desc = rows; a.best = best; a.status = status;
	a.out_logits = out; a.out_stride = vocab;
	const bool table = pick_plan(names, biases, &a);
	if (out != nullptr) return table ? pick_launch<false, true, true>(a, st) : pick_launch<false, false, true>(a, st);
	return table ? pick_launch<false, true, false>(a, st) : pick_launch<false, false, false>(a, st);
}

}  // namespace sslm

using namespace sslm;

extern "C" sslm_status sslm_b200_pick_resident(const sslm_b200_pick* call, void* stream) {
	if (!call || call->struct_size != sizeof(sslm_b200_pick)) return SSLM_INVALID_ARGUMENT;
	const sslm_b200_pick& c = *call;
	if (c.rows < 0 || c.rows > 65535 || c.vocab < 1 || c.vocab > (1 << 30) || c.num_masks < 0 || c.reserved != 0) return SSLM_INVALID_ARGUMENT;
	if (c.logits_stride < c.vocab || (c.out_logits && c.out_stride < c.vocab)) return SSLM_INVALID_ARGUMENT;
	if (c.history && (!c.history_len || c.max_history < 0 || c.max_history > kPickMaxHistory || c.history_stride < c.max_history)) return SSLM_INVALID_ARGUMENT;
	if (c.bias_tokens && (!c.bias_values || !c.bias_len || c.max_bias < 0 || c.max_bias > kPickMaxBias || c.bias_stride < c.max_bias)) return SSLM_INVALID_ARGUMENT;
	if (c.mask_page && ((!c.masks && c.num_masks > 0) || c.mask_stride < (c.vocab + 7) / 8)) return SSLM_INVALID_ARGUMENT;
	if (c.rows == 0) return SSLM_OK;      // (tensors without elements have no address)
	if (!c.logits || (!c.out_tokens && !c.out_best && !c.out_logits)) return SSLM_INVALID_ARGUMENT;
	for (const void* p : {(const void*)c.logits, (const void*)c.params, (const void*)c.history, (const void*)c.history_len, (const void*)c.bias_tokens,
	                      (const void*)c.bias_values, (const void*)c.bias_len, (const void*)c.mask_page, (const void*)c.out_tokens, (const void*)c.out_best,
	                      (const void*)c.out_logits, (const void*)c.row_status})
		if ((uintptr_t)p & 3) return SSLM_MISALIGNED_BUFFER;
	PickArgs a{};
	a.rows = c.rows; a.vocab = c.vocab;
	a.logits = c.logits; a.logits_stride = c.logits_stride;
	a.params = c.params;
	a.history = c.history; a.history_len = c.history_len; a.history_stride = c.history_stride;
	a.bias_tokens = c.bias_tokens; a.bias_values = c.bias_values; a.bias_len = c.bias_len; a.bias_stride = c.bias_stride;
	a.masks = c.masks; a.mask_stride = c.mask_stride; a.mask_page = c.mask_page; a.num_masks = c.num_masks;
	a.out_tokens = c.out_tokens; a.out_best = c.out_best; a.out_logits = c.out_logits; a.out_stride = c.out_stride;
	a.status = c.row_status;
	a.max_history = c.max_history; a.max_bias = c.max_bias;
	const int biases = c.bias_tokens ? c.max_bias : 0;
	const bool table = pick_plan((c.history ? c.max_history : 0) + biases, biases, &a);
	const auto launch = table ? (c.out_logits ? pick_launch<true, true, true> : pick_launch<true, true, false>)
	                          : (c.out_logits ? pick_launch<true, false, true> : pick_launch<true, false, false>);
	if (launch(a, (cudaStream_t)stream) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}
