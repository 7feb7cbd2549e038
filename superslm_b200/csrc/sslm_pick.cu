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
// vocabulary, which tokens the history or the biases name, with counts beside them, and which ones are allowed. The
// named tokens are few and dear (a division, a table): they are listed and dealt out one by one. All others are
// streamed past, four at a time, and cost a load, a nibble of one bitmap and a maximum; where it lies is looked up
// once, at the end. (With the named ones worked on in the stream nearly every other warp stopped for one: 256 rows
// of 151,936 with histories of 1,024 took 104 us.) Bound by the logits' bytes where rows are many, by the chain
// (lists, marks, one trip to memory, one exchange) where they are few.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/sslm_b200.h"
#include "sslm_cluster.cuh"
#include "sslm_kernels.h"

namespace sslm {

constexpr int kPickThreads = 512;
constexpr int kPickPass = 24576;            // tokens whose counts a block holds at a time (a multiple of 32)
constexpr int kPickMaxHistory = 65535;      // (a count is 16 bits)
constexpr int kPickMaxBias = 1024;

struct PickArgs {
	int rows, vocab, shift, slice;      // a row is cut over 1 << shift blocks of `slice` tokens (a multiple of 32)
	int pass;                           // tokens per pass over a slice (a multiple of 32)
	int hash;                           // places of the bias table, a power of two, or 0
	int list;                           // room for named tokens of a pass: all of it, or all that the lists can name
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

struct PickSmem {
	// bias sums [hash], bias keys [hash], counts u16 [pass + 8], allowed and named bits [pass / 32 + 2], list of named tokens u16 [list]
	static size_t bytes(int pass, int hash, int list) { return (size_t)hash * 12 + (size_t)(pass + 8) * 2 + (size_t)(pass / 32 + 2) * 8 + (size_t)list * 2; }
};

__device__ __forceinline__ unsigned long long pick_key(int32_t x, int v) {
	return x == INT32_MIN ? 0ull : (unsigned long long)((uint32_t)x ^ 0x80000000u) << 32 | (0xFFFFFFFFu - (uint32_t)v);
}

template <bool RESIDENT>
__global__ void __launch_bounds__(kPickThreads, 2) k_pick(const __grid_constant__ PickArgs a) {
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ __align__(8) unsigned long long s_bar, s_rx[16], s_warp[kPickThreads / 32];
	__shared__ int s_listed;
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.vocab;
	const int sub = 1 << a.shift, rank = (int)blockIdx.x;
	const int64_t r = blockIdx.y;
	unsigned long long* bsum = (unsigned long long*)smem;                   // [hash]
	int32_t* bkey = (int32_t*)(bsum + a.hash);                              // [hash] token, -1: free
	uint32_t* counts = (uint32_t*)(bkey + a.hash);                          // u16 pairs
	uint32_t* allow = counts + (a.pass + 8) / 2;                            // bit i: token v0 + i
	uint32_t* named = allow + a.pass / 32 + 2;
	uint16_t* list = (uint16_t*)(named + a.pass / 32 + 2);
	if (sub > 1) {
		if (t == 0 && rank == 0) {
			const int held = blockIdx.x == 0 && blockIdx.y == 0 ? a.debug_withhold : 0;
			exchange_init(cta_addr(&s_bar), (uint32_t)(sub * 8) + (held == 1 ? 4u : 0u));
			exchange_fence_init();
		}
		__syncwarp();
		cluster_arrive();      // (waited for ahead of the word that is sent)
	}
	pdl_wait();
	pdl_release();

	// ---- the row
	PickRow w{};
	int32_t code = 0;
	const int32_t* bt = nullptr;
	const int32_t* bv = nullptr;
	int32_t* out = nullptr;
	if (RESIDENT) {
		w.logits = a.logits + r * a.logits_stride;
		w.theta = 32768;
		w.extra = -1;
		if (a.params != nullptr) {
			w.theta = a.params[3 * r];
			w.presence = a.params[3 * r + 1];
			w.frequency = a.params[3 * r + 2];
			if (w.theta < 1) code = SSLM_B200_ROW_CONSTANTS;
		}
		if (a.history != nullptr) {
			w.history = a.history + r * a.history_stride;
			w.n_history = a.history_len[r];
			if (w.n_history < 0 || w.n_history > a.max_history) code = SSLM_B200_ROW_LENGTH;
		}
		if (a.bias_tokens != nullptr) {
			bt = a.bias_tokens + r * a.bias_stride;
			bv = a.bias_values + r * a.bias_stride;
			w.n_bias = a.bias_len[r];
			if (w.n_bias < 0 || w.n_bias > a.max_bias) code = SSLM_B200_ROW_LENGTH;
		}
		if (a.mask_page != nullptr) {
			const int page = a.mask_page[r];
			if (page >= a.num_masks) code = SSLM_B200_ROW_INDEX;
			else if (page >= 0) w.mask = a.masks + (int64_t)page * a.mask_stride;
		}
		if (a.out_logits != nullptr) out = a.out_logits + r * a.out_stride;
		if (rank == 0 && t == 0 && a.status != nullptr) a.status[r] = code;
	} else {
		w = a.desc[r];
		bt = w.bias_tokens;
		bv = w.bias_values;
		if (w.logits == nullptr) code = 1;      // (a row without controls)
		else if (w.extra >= 0 && rank == 0 && t == 0) const_cast<int32_t*>(w.history)[w.n_history] = w.extra;      // (its blocks count it from the descriptor)
	}
	if (code != 0) {      // (all blocks of the cluster alike)
		if (sub > 1) cluster_wait();
		return;
	}

	auto place = [&](int v) { return ((uint32_t)v * 2654435761u) >> 7 & (uint32_t)(a.hash - 1); };
	const bool listed = w.n_history > 0 || w.extra >= 0 || w.n_bias > 0;
	unsigned long long key = 0ull;      // of the named tokens and the ends
	const double inv_theta = 1.0 / (double)w.theta;
	const int s0 = min(V, rank * a.slice), s1 = min(V, s0 + a.slice);
	// four neighbouring tokens of the row lie in one aligned 16-byte word; mis: tokens by which the row's first is off
	const int mis = (int)(((uintptr_t)w.logits >> 2) & 3);
	const int mis_out = (int)(((uintptr_t)out >> 2) & 3);
	constexpr int U = 5, kStride = 4 * kPickThreads;
	for (int v0 = s0; v0 < s1; v0 += a.pass) {
		const int v1 = min(s1, v0 + a.pass), n = v1 - v0, words = (n + 31) / 32;
		// whole aligned words of four tokens, `first` to `last`; the ends of the pass one by one
		const int first = min(v1, v0 + ((4 - ((v0 + mis) & 3)) & 3)), last = first + ((v1 - first) & ~3);
		const int32_t* mine = w.logits + first + 4 * t;
		const int turns = first + 4 * t < last ? (last - first - 4 * t + kStride - 1) / kStride : 0;      // this thread's words
		int4 x[U];      // (on their way while the marks are made)
#pragma unroll
		for (int u = 0; u < U; ++u)
			if (u < turns) x[u] = __ldcs((const int4*)(mine + u * kStride));
		// ---- marks and counts of tokens v0 .. v1
		for (int i = t; i < words + 2; i += kPickThreads) {
			uint32_t bits = 0;
			const int left = n - i * 32;
			if (left > 0) {
				bits = left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u;
				if (w.mask != nullptr) {      // (v0 is a multiple of 32; a page has ceil(V / 8) bytes and any address)
					const uint8_t* m = w.mask + (v0 >> 3) + 4 * i;
					uint32_t page = 0;
					if (left >= 32 && ((uintptr_t)m & 3) == 0) page = *(const uint32_t*)m;
					else
						for (int j = 0; j < min(4, (left + 7) >> 3); ++j) page |= (uint32_t)m[j] << (8 * j);
					bits &= page;
				}
			}
			allow[i] = bits;
			named[i] = 0u;
		}
		if (listed) {
			for (int i = t; i < (n + 8) / 8; i += kPickThreads) ((int4*)counts)[i] = make_int4(0, 0, 0, 0);
			for (int i = t; i < a.hash; i += kPickThreads) {
				bkey[i] = -1;
				bsum[i] = 0ull;
			}
			if (t == 0) s_listed = 0;
			__syncthreads();
			auto name = [&](uint32_t i) {      // the first to name a token enters it into the list
				if ((atomicOr(&named[i >> 5], 1u << (i & 31)) >> (i & 31) & 1u) == 0u) list[atomicAdd(&s_listed, 1)] = (uint16_t)i;
			};
			auto seen = [&](int v) {
				const uint32_t i = (uint32_t)(v - v0);
				if (i >= (uint32_t)n) return;
				atomicAdd(&counts[i >> 1], 1u << (16 * (i & 1)));
				name(i);
			};
			{      // (ids of any alignment: single ones up to the first 16-byte word, then words)
				const int head = min(w.n_history, (int)((4 - (((uintptr_t)w.history >> 2) & 3)) & 3)), whole = (w.n_history - head) >> 2;
				if (t < head) seen(w.history[t]);
				const int4* ids = (const int4*)(w.history + head);
#pragma unroll 2
				for (int i = t; i < whole; i += kPickThreads) {
					const int4 id = ids[i];
					seen(id.x);
					seen(id.y);
					seen(id.z);
					seen(id.w);
				}
				const int tail = head + 4 * whole + t;
				if (tail < w.n_history) seen(w.history[tail]);
			}
			if (t == 0 && w.extra >= 0) seen(w.extra);
			for (int i = t; i < w.n_bias; i += kPickThreads) {
				const int v = bt[i];
				const uint32_t at = (uint32_t)(v - v0);
				if (at >= (uint32_t)n) continue;
				uint32_t h = place(v);
				for (;;) {      // (at least half of the places stay free)
					const int was = atomicCAS(&bkey[h], -1, v);
					if (was == -1 || was == v) break;
					h = (h + 1) & (uint32_t)(a.hash - 1);
				}
				atomicAdd(&bsum[h], (unsigned long long)(long long)bv[i]);
				name(at);
			}
			__syncthreads();
			// ---- the named tokens
#pragma unroll 2
			for (int k = t; k < s_listed; k += kPickThreads) {
				const int i = list[k], v = v0 + i;
				int32_t y = w.logits[v];
				if (y != INT32_MIN) {
					long long z = y;
					const uint32_t cnt = counts[i >> 1] >> (16 * (i & 1)) & 0xFFFFu;
					if (cnt != 0u) {
						if (z > 0) {      // floor(2^15 z / theta): a quotient in doubles, off by one at most, settled by its remainder
							const long long num = z << 15;
							long long q = (long long)((double)num * inv_theta);
							const long long rem = num - q * (long long)w.theta;
							z = q + (rem >= (long long)w.theta ? 1 : 0) - (rem < 0 ? 1 : 0);
						} else {
							z = -((-z * (long long)w.theta) >> 15);
						}
						z -= (long long)w.presence + (long long)w.frequency * (long long)cnt;
					}
					if (w.n_bias > 0) {
						uint32_t h = place(v);
						while (bkey[h] != v && bkey[h] != -1) h = (h + 1) & (uint32_t)(a.hash - 1);
						if (bkey[h] == v) z += (long long)bsum[h];
					}
					y = (int32_t)max(-2147483647ll, min(2147483647ll, z));
				}
				if ((allow[i >> 5] >> (i & 31) & 1u) == 0u) y = INT32_MIN;
				key = max(key, pick_key(y, v));
				if (out != nullptr) out[v] = y;
			}
		} else {
			__syncthreads();
		}
		// ---- all others
		auto one = [&](int v) {
			const int i = v - v0;
			if ((named[i >> 5] >> (i & 31) & 1u) != 0u) return;
			const int32_t y = (allow[i >> 5] >> (i & 31) & 1u) != 0u ? w.logits[v] : INT32_MIN;
			key = max(key, pick_key(y, v));
			if (out != nullptr) out[v] = y;
		};
		if (t < first - v0) one(v0 + t);
		if (t < v1 - last) one(last + t);
		// the words of a thread lie a multiple of 32 tokens apart: their bits at one place of their bitmap words
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
		int top_at = 0;      // the word that has it first
		for (int k0 = 0; k0 < turns; k0 += U) {
#pragma unroll
			for (int u = 0; u < U; ++u) {
				const int k = k0 + u;
				if (k >= turns) break;
				const int4 q = x[u];
				if (k + U < turns) x[u] = __ldcs((const int4*)(mine + (k + U) * kStride));
				const uint32_t nm = listed ? nibble(named, k) : 0u;
				int32_t y[4];
				words_of(q, nibble(allow, k) & ~nm, y);
				const int32_t m = max(max(y[0], y[1]), max(y[2], y[3]));
				if (m > top) {
					top = m;
					top_at = k;
				}
				if (out != nullptr) {
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
		}
		if (top != INT32_MIN) {      // (in place, the word reads as it was but for what the bitmaps leave out)
			int32_t y[4];
			words_of(*(const int4*)(mine + top_at * kStride), nibble(allow, top_at) & ~(listed ? nibble(named, top_at) : 0u), y);
			const int j = y[0] == top ? 0 : (y[1] == top ? 1 : (y[2] == top ? 2 : 3));
			key = max(key, pick_key(top, first + 4 * t + top_at * kStride + j));
		}
		__syncthreads();      // the tables may be overwritten
	}
	// ---- the row's largest key: larger values first, then lower indices
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
	if (lane == 0) s_warp[warp] = key;
	__syncthreads();
	if (warp != 0) {
		if (sub > 1) cluster_wait();
		return;
	}
	key = lane < kPickThreads / 32 ? s_warp[lane] : 0ull;
#pragma unroll
	for (int o = 8; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
	bool ok = true;
	if (sub > 1) {
		cluster_wait();      // (the first block runs)
		if (lane == 0) exchange_send(&s_rx[rank], cta_addr(&s_bar), 0u, key);
		if (rank != 0) return;      // (nothing is sent to it)
		ok = exchange_wait(cta_addr(&s_bar));
		key = lane < sub ? s_rx[lane] : 0ull;
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
		exchange_leave(cta_addr(&s_bar), 1);
	}
}

namespace {

// Blocks per row: slices of at least 4,096 tokens, eight blocks at most.
// names: how many tokens the lists of a row can name.
void pick_plan(int vocab, int names, int bias, PickArgs* a) {
	a->shift = 0;
	while (a->shift < 3 && vocab >> (a->shift + 1) >= 4096) ++a->shift;
	if (a->shift == 3 && a->rows * 16 <= sm_count() && vocab >= 16 * 4096) a->shift = 4;      // (few rows: the chain is shorter)
	a->slice = (((vocab + (1 << a->shift) - 1) >> a->shift) + 31) & ~31;
	a->pass = std::min(a->slice, kPickPass);
	a->list = std::min(a->pass, names);
	a->hash = 0;
	if (bias > 0) {
		a->hash = 16;
		while (a->hash < 2 * bias) a->hash *= 2;
	}
}

template <bool RESIDENT>
cudaError_t pick_launch(PickArgs a, cudaStream_t st) {
	static PerDeviceOnce once;
	cudaError_t e = once_per_device(once, [&] {
		cudaError_t x = cudaFuncSetAttribute(k_pick<RESIDENT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
		if (x != cudaSuccess) return x;
		return cudaFuncSetAttribute(k_pick<RESIDENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PickSmem::bytes(kPickPass, 2 * kPickMaxBias, kPickPass));
	});
	if (e != cudaSuccess) return e;
	a.debug_withhold = a.shift > 0 ? exchange_debug_take(kExchangePick) : 0;
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3(1u << a.shift, a.rows);
	cfg.blockDim = dim3(kPickThreads);
	cfg.dynamicSmemBytes = PickSmem::bytes(a.pass, a.hash, a.list);
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
	return cudaLaunchKernelEx(&cfg, k_pick<RESIDENT>, a);
}

}  // namespace
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
	if (!c.out_tokens && !c.out_best && !c.out_logits) return SSLM_INVALID_ARGUMENT;
	if (c.rows == 0) return SSLM_OK;
	if (!c.logits) return SSLM_INVALID_ARGUMENT;
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
	pick_plan(c.vocab, (c.history ? c.max_history : 0) + (c.bias_tokens ? c.max_bias : 0), c.bias_tokens ? c.max_bias : 0, &a);
	if (pick_launch<true>(a, (cudaStream_t)stream) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}
