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
// One pass over the logits. A row is cut over the blocks of a cluster; a block first builds, for its slice of
// the vocabulary, two bitmaps in shared memory -- which tokens are allowed, which ones the history or the biases
// name -- and 16-bit counts beside them, then streams its logits. Four neighbouring tokens that nothing names,
// nearly all of them, cost a load, two bitmap words and a maximum. Bound by the logits' bytes where rows are many, by
// the chain (lists, bitmaps, one trip to memory, one exchange) where they are few.
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
	// counts u16 [pass + 8], allowed bits [pass / 32 + 2], named bits [pass / 32 + 2], bias keys [hash], bias sums [hash]
	static size_t bytes(int pass, int hash) { return (size_t)hash * 12 + (size_t)(pass + 8) * 2 + (size_t)(pass / 32 + 2) * 8; }
};

__device__ __forceinline__ unsigned long long pick_key(int32_t x, int v) {
	return x == INT32_MIN ? 0ull : (unsigned long long)((uint32_t)x ^ 0x80000000u) << 32 | (0xFFFFFFFFu - (uint32_t)v);
}

template <bool RESIDENT>
__global__ void __launch_bounds__(kPickThreads) k_pick(const __grid_constant__ PickArgs a) {
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ __align__(8) unsigned long long s_bar, s_rx[16], s_warp[kPickThreads / 32];
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.vocab;
	const int sub = 1 << a.shift, rank = (int)blockIdx.x;
	const int64_t r = blockIdx.y;
	unsigned long long* bsum = (unsigned long long*)smem;                   // [hash]
	int32_t* bkey = (int32_t*)(bsum + a.hash);                              // [hash] token, -1: free
	uint32_t* counts = (uint32_t*)(bkey + a.hash);                          // u16 pairs
	uint32_t* allow = counts + (a.pass + 8) / 2;                            // bit i: token v0 + i
	uint32_t* named = allow + a.pass / 32 + 2;
	if (sub > 1) {
		if (t == 0 && rank == 0) {
			const int held = blockIdx.x == 0 && blockIdx.y == 0 ? a.debug_withhold : 0;
			exchange_init(cta_addr(&s_bar), (uint32_t)(sub * 8) + (held == 1 ? 4u : 0u));
			exchange_fence_init();
		}
		cluster_arrive();
		cluster_wait();
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
	if (code != 0) return;      // (all blocks of the cluster alike)

	const bool listed = w.n_history > 0 || w.extra >= 0 || w.n_bias > 0;
	int32_t top = INT32_MIN;
	int top_at = 0;
	const int s0 = min(V, rank * a.slice), s1 = min(V, s0 + a.slice);
	// four neighbouring tokens of the row lie in one aligned 16-byte word; mis: tokens by which the row's first is off
	const int mis = (int)(((uintptr_t)w.logits >> 2) & 3);
	const int mis_out = (int)(((uintptr_t)out >> 2) & 3);
	for (int v0 = s0; v0 < s1; v0 += a.pass) {
		const int v1 = min(s1, v0 + a.pass), n = v1 - v0, words = (n + 31) / 32;
		// ---- bitmaps and counts of tokens v0 .. v1
		for (int i = t; i < words + 2; i += kPickThreads) {
			uint32_t bits = 0;
			const int left = n - i * 32;
			if (left > 0) {
				bits = left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u;
				if (w.mask != nullptr) {      // (v0 is a multiple of 32; a page has ceil(V / 8) bytes and any address)
					const uint8_t* m = w.mask + (v0 >> 3) + 4 * i;
					const int nbytes = min(4, (left + 7) >> 3);
					uint32_t page = 0;
					for (int j = 0; j < nbytes; ++j) page |= (uint32_t)m[j] << (8 * j);
					bits &= page;
				}
			}
			allow[i] = bits;
			named[i] = 0u;
		}
		if (listed) {
			for (int i = t; i < (n + 8) / 2; i += kPickThreads) counts[i] = 0u;
			for (int i = t; i < a.hash; i += kPickThreads) {
				bkey[i] = -1;
				bsum[i] = 0ull;
			}
		}
		__syncthreads();
		if (listed) {
			auto seen = [&](int v) {
				const uint32_t i = (uint32_t)(v - v0);
				if (i >= (uint32_t)n) return;
				atomicAdd(&counts[i >> 1], 1u << (16 * (i & 1)));
				atomicOr(&named[i >> 5], 1u << (i & 31));
			};
			for (int i = t; i < w.n_history; i += kPickThreads) seen(w.history[i]);
			if (t == 0 && w.extra >= 0) seen(w.extra);
			for (int i = t; i < w.n_bias; i += kPickThreads) {
				const int v = bt[i];
				const uint32_t at = (uint32_t)(v - v0);
				if (at >= (uint32_t)n) continue;
				uint32_t h = ((uint32_t)v * 2654435761u) >> 7 & (uint32_t)(a.hash - 1);
				for (;;) {      // (at least half of the places stay free)
					const int was = atomicCAS(&bkey[h], -1, v);
					if (was == -1 || was == v) break;
					h = (h + 1) & (uint32_t)(a.hash - 1);
				}
				atomicAdd(&bsum[h], (unsigned long long)(long long)bv[i]);
				atomicOr(&named[at >> 5], 1u << (at & 31));
			}
			__syncthreads();
		}
		// ---- the logits
		auto changed = [&](int32_t x32, int v) {      // a token that a list names
			const int i = v - v0;
			long long x = x32;
			const uint32_t cnt = counts[i >> 1] >> (16 * (i & 1)) & 0xFFFFu;
			if (cnt != 0u) {
				x = x > 0 ? (x << 15) / w.theta : -((-x * (long long)w.theta) >> 15);
				x -= (long long)w.presence + (long long)w.frequency * (long long)cnt;
			}
			if (w.n_bias > 0) {
				uint32_t h = ((uint32_t)v * 2654435761u) >> 7 & (uint32_t)(a.hash - 1);
				while (bkey[h] != v && bkey[h] != -1) h = (h + 1) & (uint32_t)(a.hash - 1);
				if (bkey[h] == v) x += (long long)bsum[h];
			}
			return (int32_t)max(-2147483647ll, min(2147483647ll, x));
		};
		auto take = [&](int32_t x, int v) {
			if (x > top) {
				top = x;
				top_at = v;
			}
		};
		auto one = [&](int32_t x, int v) {
			const int i = v - v0;
			if (x != INT32_MIN && (named[i >> 5] >> (i & 31) & 1u) != 0u) x = changed(x, v);
			if ((allow[i >> 5] >> (i & 31) & 1u) == 0u) x = INT32_MIN;
			take(x, v);
			if (out != nullptr) out[v] = x;
		};
		// whole aligned words of the pass, and its ends one by one
		const int first = v0 + ((4 - ((v0 + mis) & 3)) & 3), last = first + (v1 > first ? (v1 - first) & ~3 : 0);
		if (t < min(first, v1) - v0) one(w.logits[v0 + t], v0 + t);
		constexpr int U = 4;
		for (int b = first + 4 * t; b < last; b += 4 * U * kPickThreads) {
			int4 x[U];
#pragma unroll
			for (int u = 0; u < U; ++u) {
				const int v = b + 4 * u * kPickThreads;
				if (v < last) x[u] = __ldcs((const int4*)(w.logits + v));
			}
#pragma unroll
			for (int u = 0; u < U; ++u) {
				const int v = b + 4 * u * kPickThreads, i = v - v0;
				if (v >= last) break;
				const uint32_t al = __funnelshift_r(allow[i >> 5], allow[(i >> 5) + 1], i & 31) & 15u;
				const uint32_t nm = __funnelshift_r(named[i >> 5], named[(i >> 5) + 1], i & 31) & 15u;
				int32_t y[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
				if (nm != 0u) {
#pragma unroll
					for (int j = 0; j < 4; ++j)
						if ((nm >> j & 1u) != 0u && y[j] != INT32_MIN) y[j] = changed(y[j], v + j);
				}
				if (al != 15u) {
#pragma unroll
					for (int j = 0; j < 4; ++j) y[j] = (al >> j & 1u) != 0u ? y[j] : INT32_MIN;
				}
				if (max(max(y[0], y[1]), max(y[2], y[3])) > top) {
#pragma unroll
					for (int j = 0; j < 4; ++j) take(y[j], v + j);
				}
				if (out != nullptr) {
					if (mis_out == mis) {
						__stcs((int4*)(out + v), make_int4(y[0], y[1], y[2], y[3]));
					} else {
#pragma unroll
						for (int j = 0; j < 4; ++j) out[v + j] = y[j];
					}
				}
			}
		}
		const int tail = max(first, last);
		if (tail < v1 && t < v1 - tail) one(w.logits[tail + t], tail + t);
		__syncthreads();      // the tables may be overwritten
	}
	// ---- the row's largest key: larger values first, then lower indices
	unsigned long long key = pick_key(top, top_at);
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
	if (lane == 0) s_warp[warp] = key;
	__syncthreads();
	if (warp != 0) return;
	key = lane < kPickThreads / 32 ? s_warp[lane] : 0ull;
#pragma unroll
	for (int o = 8; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
	bool ok = true;
	if (sub > 1) {
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
void pick_plan(int vocab, int bias, PickArgs* a) {
	a->shift = 0;
	while (a->shift < 3 && vocab >> (a->shift + 1) >= 4096) ++a->shift;
	a->slice = (((vocab + (1 << a->shift) - 1) >> a->shift) + 31) & ~31;
	a->pass = std::min(a->slice, kPickPass);
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
		return cudaFuncSetAttribute(k_pick<RESIDENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PickSmem::bytes(kPickPass, 2 * kPickMaxBias));
	});
	if (e != cudaSuccess) return e;
	a.debug_withhold = a.shift > 0 ? exchange_debug_take(kExchangePick) : 0;
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3(1u << a.shift, a.rows);
	cfg.blockDim = dim3(kPickThreads);
	cfg.dynamicSmemBytes = PickSmem::bytes(a.pass, a.hash);
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
	pick_plan(c.vocab, c.bias_tokens ? c.max_bias : 0, &a);
	if (pick_launch<true>(a, (cudaStream_t)stream) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}
