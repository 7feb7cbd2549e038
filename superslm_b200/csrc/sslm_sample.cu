// A token drawn from int32 logits: temperature, top-k, top-p, min-p and a given random number, in integers throughout.
//
// Per row, over the tokens v whose logit x_v is not INT32_MIN, d_v = max x - x_v:
//   w_v = 2^31 2^-(d_v slope)      slope = m / 2^(24 + e) octaves a logit unit; t = floor(d m / 2^e) has 24 bits behind the point, its whole
//                                  part shifts, and 2^-f of the rest is a polynomial of degree 4 (Horner, high halves of 32-bit products)
//   in the order of falling logits, equal ones by rising index: the first top_k; of their sum S those before which less than
//   floor(S top_p / 2^30) lies; of them those with w >= 2 min_p (the largest weight is 2^31)
//   the token: the lowest v up to which more than floor(sum u / 2^31) of the kept weights lies, by index
// All sums are of integers, so no order of adding changes one.
//
// The polynomial is the fit of the smallest largest relative error (3.3e-6) with the values 1 and 1/2 at the ends, its last coefficients rounded
// up by less than one part in 10^7, which leaves it falling from octave to octave too (checked for all 2^24 arguments): w falls with d.
//
// Two passes over the logits. The first finds the row's maximum and a bound that is likely to lie below what is kept and above nearly all else: the
// least of the maxima of some hundred groups of threads. g groups leave about g ln g tokens above it (and g at least). The second pass
// lists these tokens, a few hundred to a few thousand, and adds up all weights where top-p needs that. What is kept is then cut and drawn
// from the list by counting into 2,048 places. Where the list does not reach far enough (its weights, or its length, tell) or overflows, the
// same counting goes over the whole row. Rows without top-k and top-p need no list: sums of 128 neighbouring tokens are enough to find
// the token.
//
// A row is cut over the blocks of a cluster while rows are few; they exchange maxima and sums, and send their lists to the first one.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/sslm_b200.h"
#include "sslm_cluster.cuh"
#include "sslm_kernels.h"

namespace sslm {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kList = 8192;                   // tokens of a row's list
constexpr int kPlaces = 2048;                 // that a selection counts into
constexpr int kIndexBits = 20;                // of a token
constexpr int kMostVocab = 1 << kIndexBits;
constexpr int kMostSlice = (kPlaces - 2) * 128 & ~127;      // a sum for every 128 tokens, and for the ends
constexpr uint32_t kLate = 0xFFFFFFFFu;

struct SampleArgs {
	int rows, vocab, shift, slice;      // a row is cut over 1 << shift blocks of `slice` tokens (a multiple of 128)
	int keep;                           // the block's logits stay in shared memory
	// a caller's tensors
	const int32_t* logits;
	int64_t logits_stride;
	const int32_t *params, *draws;
	int32_t *out_tokens, *out_kept, *status;
	int64_t* out_mass;
	// rows of an engine call
	const SampleRow* desc;
	const Scale* scales;                // of the rows that the head multiplied
	unsigned long long* best;
	int debug_withhold;
};

struct Row {
	const int32_t* logits;
	uint32_t slope, cut, draw;
	int top_k, code, layer;
	uint32_t top_p, min_p;
};

// ---- weights
__device__ __forceinline__ uint32_t weight_of(uint32_t d, uint32_t most, uint32_t slope, uint32_t cut) {
	const uint32_t t = (uint32_t)(((unsigned long long)d * slope) >> cut);      // (below 2^29 up to `most`)
	const uint32_t f = t << 8;
	uint32_t p = 14555373u;
	p = 114090822u - __umulhi(f, p);
	p = 514119776u - __umulhi(f, p);
	p = 1488326151u - __umulhi(f, p);
	p = 2147483648u - __umulhi(f, p);
	return d <= most ? p >> (t >> 24) : 0u;
}
// the largest d with a weight: d slope < 2^(29 + cut)
__device__ __forceinline__ uint32_t farthest(uint32_t slope, uint32_t cut) {
	if (slope == 0u || cut >= 34u) return 0xFFFFFFFFu;      // (d slope is below 2^63)
	const unsigned long long q = ((1ull << (29 + cut)) - 1ull) / slope;
	return q > 0xFFFFFFFFull ? 0xFFFFFFFFu : (uint32_t)q;
}
// floor(total part / 2^bits), part <= 2^bits
__device__ __forceinline__ unsigned long long share_of(unsigned long long total, uint32_t part, int bits) {
	const unsigned long long lo = total * part, hi = __umul64hi(total, part);
	return lo >> bits | hi << (64 - bits);
}

// ---- block-wide sums and maxima; s: kWarps words
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
	return v;
}
__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, unsigned long long* s) {
	v = warp_sum(v);
	__syncthreads();
	if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
	__syncthreads();
	unsigned long long all = 0;
#pragma unroll
	for (int i = 0; i < kWarps; ++i) all += s[i];
	return all;
}

// ---- selection: of elements with keys that differ and weights, the first one, by rising keys, up to which (itself included) more than
// `target` of the weights lies. The elements are counted into 2,048 places by their keys' leading bits, the place that holds the one looked for
// likewise, and so on until a place has at most 32.
struct Place { unsigned long long* sum; uint32_t* count; };      // [kPlaces] each
struct SelectSmem {
	unsigned long long key[32], weight[32], scan[kWarps], target;
	uint32_t place, count, n;
	unsigned long long found;
};
// each(f): f(key, weight) for this thread's elements. bits: all keys are below 2^bits. The sum of all weights is above target.
template <typename Each>
__device__ __noinline__ unsigned long long select_key(const Each& each, int bits, unsigned long long target, Place at, SelectSmem& s) {
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
	unsigned long long low = 0;
	for (;;) {
		const int down = max(0, bits - 11);
		for (int i = t; i < kPlaces; i += kThreads) {
			at.sum[i] = 0ull;
			at.count[i] = 0u;
		}
		if (t == 0) s.n = 0u;
		__syncthreads();
		each([&](unsigned long long key, uint32_t w) {
			const unsigned long long i = (key - low) >> down;
			if (key >= low && i < (unsigned long long)kPlaces) {
				atomicAdd(&at.sum[i], (unsigned long long)w);
				atomicAdd(&at.count[i], 1u);
			}
		});
		__syncthreads();
		// sums up to each place: four places a thread
		unsigned long long v[4], mine = 0;
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			v[j] = at.sum[4 * t + j];
			mine += v[j];
		}
		unsigned long long upto = mine;
#pragma unroll
		for (int o = 1; o < 32; o *= 2) {
			const unsigned long long z = __shfl_up_sync(0xffffffffu, upto, o);
			if (lane >= o) upto += z;
		}
		if (lane == 31) s.scan[warp] = upto;
		__syncthreads();
		unsigned long long before = upto - mine;
		for (int i = 0; i < warp; ++i) before += s.scan[i];
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			if (before <= target && target < before + v[j]) {      // (one thread's one place)
				s.place = 4 * t + j;
				s.count = at.count[4 * t + j];
				s.target = target - before;
			}
			before += v[j];
		}
		__syncthreads();
		low += (unsigned long long)s.place << down;
		target = s.target;
		const uint32_t n = s.count;
		if (n <= 32u || down == 0) {
			each([&](unsigned long long key, uint32_t w) {
				if (key >= low && ((key - low) >> down) == 0ull) {
					const uint32_t i = atomicAdd(&s.n, 1u);
					if (i < 32u) {
						s.key[i] = key;
						s.weight[i] = w;
					}
				}
			});
			__syncthreads();
			if (warp == 0) {
				const unsigned long long key = lane < n ? s.key[lane] : ~0ull, w = lane < n ? s.weight[lane] : 0ull;
				unsigned long long less = 0;
				for (int i = 0; i < 32; ++i) {
					const unsigned long long k = __shfl_sync(0xffffffffu, key, i), x = __shfl_sync(0xffffffffu, w, i);
					if (k < key) less += x;
				}
				if (lane < n && less <= target && target < less + w) s.found = key;
			}
			__syncthreads();
			return s.found;
		}
		bits = down;
	}
}

struct SampleSmem {
	// keys of the list [kList], sums [kPlaces], counts [kPlaces], the block's logits [slice] if they are kept
	static size_t bytes(int keep, int slice) { return (size_t)kList * 8 + (size_t)kPlaces * 12 + (keep ? (size_t)slice * 4 + 16 : 0); }
};

template <bool RESIDENT, bool KEEP>
__global__ void __launch_bounds__(kThreads, KEEP ? 1 : 2) k_sample(const __grid_constant__ SampleArgs a) {
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ __align__(8) unsigned long long s_bar[3], s_sum[16], s_scan[kWarps];
	__shared__ int2 s_top[16], s_warp[kWarps];
	__shared__ uint32_t s_count[16], s_n;
	__shared__ Row s_row;
	__shared__ SelectSmem s_select;
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.vocab;
	const int sub = 1 << a.shift, rank = (int)blockIdx.x;
	const int64_t r = blockIdx.y;
	unsigned long long* list = (unsigned long long*)smem;
	const Place places{list + kList, (uint32_t*)(list + kList + kPlaces)};
	int4* kept = (int4*)(places.count + kPlaces);
	const int held = (blockIdx.x | blockIdx.y) == 0 ? a.debug_withhold : 0;
	if (t == 0) {
		if (sub > 1) {
			exchange_init(cta_addr(&s_bar[0]), (uint32_t)(sub * 8) + (held == 1 ? 4u : 0u));
			exchange_init(cta_addr(&s_bar[1]), (uint32_t)(sub * 12) + (held == 2 ? 4u : 0u));
			ring_init(cta_addr(&s_bar[2]), 1);      // (armed when the lists' lengths are known)
			exchange_fence_init();
		}
		s_n = 0u;
	}
	if (sub > 1) {
		__syncwarp();
		cluster_arrive();
	}
	pdl_wait();
	pdl_release();

	// ---- the row
	if (t == 0) {
		Row x{};
		if (RESIDENT) {
			x.logits = a.logits + r * a.logits_stride;
			const int32_t* p = a.params + 5 * r;
			const int32_t slope = p[0], cut = p[1], top_k = p[2], top_p = p[3], min_p = p[4], draw = a.draws[r];
			if (slope < 0 || cut < 0 || cut > 63 || top_k < 0 || top_p < 1 || top_p > (1 << 30) || min_p < 0 || min_p > (1 << 30) || draw < 0) x.code = SSLM_B200_ROW_CONSTANTS;
			x.slope = (uint32_t)slope; x.cut = (uint32_t)cut; x.draw = (uint32_t)draw;
			x.top_k = top_k; x.top_p = (uint32_t)top_p; x.min_p = (uint32_t)min_p;
			if (rank == 0 && a.status != nullptr) a.status[r] = x.code;
		} else {
			const SampleRow d = a.desc[r];
			x.logits = d.logits;
			if (d.logits == nullptr) {
				x.code = 1;      // (a row that is not sampled)
			} else {
				// octaves a logit unit: the sequence's constant times the scale of the row that the head multiplied
				const Scale s = combine(Scale{d.slope_m, d.slope_e}, a.scales[r]);
				const int64_t cut = -(s.e + 24);
				x.slope = cut < 0 ? 1u << 30 : (cut > 94 ? 0u : (uint32_t)s.m >> (cut > 63 ? (int)cut - 63 : 0));      // (64 octaves a unit are as good as more)
				x.cut = (uint32_t)max((int64_t)0, min((int64_t)63, cut));
				x.draw = d.draw;
				x.top_k = d.top_k; x.top_p = d.top_p; x.min_p = d.min_p;
				x.layer = d.layer;
			}
		}
		s_row = x;
	}
	__syncthreads();
	const Row w = s_row;
	if (w.code != 0) {      // (all blocks of the cluster alike)
		if (sub > 1) cluster_wait();
		return;
	}
	const int s0 = min(V, rank * a.slice), s1 = min(V, s0 + a.slice);
	// four neighbouring tokens lie in one aligned 16-byte word: whole words from `first` to `last`, the ends token by token
	const int mis = (int)(((uintptr_t)w.logits >> 2) & 3);
	const int first = min(s1, s0 + ((4 - ((s0 + mis) & 3)) & 3)), words = (s1 - first) >> 2, last = first + 4 * words;
	const int4* from = (const int4*)(w.logits + first);
	const int heads = first - s0, tails = s1 - last;
	const int end = t < heads ? s0 + t : (t >= 4 && t - 4 < tails ? last + t - 4 : -1);      // the token of the ends that is this thread's
	const int32_t end_x = end >= 0 ? w.logits[end] : INT32_MIN;

	// ---- the maximum, and the least of the groups' maxima
	int32_t top = end_x;
	constexpr int U = 8;
#pragma unroll 1
	for (int k = t; k < words; k += U * kThreads) {
		int4 q[U];
#pragma unroll
		for (int u = 0; u < U; ++u)
			if (k + u * kThreads < words) q[u] = __ldcg(from + k + u * kThreads);
#pragma unroll
		for (int u = 0; u < U; ++u)
			if (k + u * kThreads < words) {
				if (KEEP) kept[k + u * kThreads] = q[u];
				top = max(top, max(max(q[u].x, q[u].y), max(q[u].z, q[u].w)));
			}
	}
	const bool cuts = w.top_k > 0 || w.top_p < (1u << 30);
	int32_t least = INT32_MAX;
	if (cuts) {
		const int wanted = w.top_k > 0 && w.top_k <= 64 ? 128 : 512, lanes = max(1, min(32, sub * kThreads / wanted));
		least = t < words || end >= 0 ? top : INT32_MIN;
		for (int o = 1; o < lanes; o *= 2) least = max(least, __shfl_xor_sync(0xffffffffu, least, o));
		// (threads without a token count only where their whole group has none)
		const uint32_t has = __ballot_sync(0xffffffffu, t < words || end >= 0);
		const uint32_t group = lanes == 32 ? 0xFFFFFFFFu : ((1u << lanes) - 1u) << (lane & ~(lanes - 1));
		if ((has & group) == 0u) least = INT32_MAX;
	}
	{
		const int32_t m = __reduce_max_sync(0xffffffffu, top), l = __reduce_min_sync(0xffffffffu, least);
		if (lane == 0) s_warp[warp] = make_int2(m, l);
	}
	__syncthreads();
	{
		const int2 x = s_warp[lane & (kWarps - 1)];
		top = __reduce_max_sync(0xffffffffu, x.x);
		least = __reduce_min_sync(0xffffffffu, x.y);
		if (top == INT32_MIN) least = INT32_MAX;      // (nothing is allowed here)
	}
	bool late = false;
	if (sub > 1) {
		cluster_wait();      // (all blocks run)
		if (t < sub) exchange_send(&s_top[rank], cta_addr(&s_bar[0]), (uint32_t)t, make_int2(top, least));
		late = !exchange_wait(cta_addr(&s_bar[0]));
		const int2 x = s_top[lane & (sub - 1)];
		top = __reduce_max_sync(0xffffffffu, x.x);
		least = __reduce_min_sync(0xffffffffu, x.y);
	}
	late = __syncthreads_or(late) != 0;
	const bool none = top == INT32_MIN;

	// ---- the second pass
	const uint32_t most = farthest(w.slope, w.cut), floor_w = max(1u, 2u * w.min_p);
	const uint32_t reach = least == INT32_MIN ? 0xFFFFFFFFu : (uint32_t)top - (uint32_t)max(least, INT32_MIN + 1), far = min(reach, most);      // the list's farthest
	unsigned long long sum = 0;
	uint32_t count = 0;
	auto word = [&](int k) { return KEEP ? kept[k] : __ldcg(from + k); };
	if (!late && !none) {
		if (!cuts) {
			// sums of what is kept of 128 neighbouring tokens: places 1 .. , the ends at 0 and behind
			const int steps = (words + 31) / 32;
			auto keep_of = [&](int32_t x) {
				const uint32_t g = weight_of((uint32_t)top - (uint32_t)x, most, w.slope, w.cut);
				const bool yes = x != INT32_MIN && g >= floor_w;
				count += yes ? 1u : 0u;
				return yes ? g : 0u;
			};
			if (t < 2) places.sum[t == 0 ? 0 : steps + 1] = 0ull;
			__syncthreads();
			if (end >= 0) {
				const uint32_t g = keep_of(end_x);
				sum += g;
				atomicAdd(&places.sum[t < 4 ? 0 : steps + 1], (unsigned long long)g);
			}
#pragma unroll 4
			for (int k = t; k - lane < words; k += kThreads) {
				unsigned long long g = 0;
				if (k < words) {
					const int4 q = word(k);
					g = (unsigned long long)keep_of(q.x) + keep_of(q.y) + keep_of(q.z) + keep_of(q.w);
				}
				sum += g;
				const uint32_t high = __reduce_add_sync(0xffffffffu, (uint32_t)(g >> 16)), low = __reduce_add_sync(0xffffffffu, (uint32_t)g & 0xFFFFu);
				if (lane == 0) places.sum[1 + (k >> 5)] = ((unsigned long long)high << 16) + low;
			}
		} else {
			const bool all = w.top_k == 0;      // all weights are added up
			auto look = [&](int32_t x, int v) {
				const uint32_t d = (uint32_t)top - (uint32_t)x;
				if (all && x != INT32_MIN) sum += weight_of(d, most, w.slope, w.cut);
				const bool yes = x != INT32_MIN && d <= far;
				const uint32_t who = __ballot_sync(0xffffffffu, yes);
				if (who == 0u) return;
				uint32_t at = 0;
				if (lane == 0) at = atomicAdd(&s_n, __popc(who));
				at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
				if (yes && at < (uint32_t)kList) list[at] = (unsigned long long)d << kIndexBits | (uint32_t)v;
			};
			if (warp == 0) look(end_x, end);
#pragma unroll 4
			for (int k = t; k - lane < words; k += kThreads) {
				const int4 q = k < words ? word(k) : make_int4(INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN);
				const int v = first + 4 * k;
				look(q.x, v);
				look(q.y, v + 1);
				look(q.z, v + 2);
				look(q.w, v + 3);
			}
		}
	}
	sum = block_sum(sum, s_scan);
	if (!cuts) count = (uint32_t)block_sum(count, s_scan);
	else count = s_n;
	int owner = 0;                          // the block that finds the token
	unsigned long long mark = 0;            // and how much of what is kept lies before what it looks for
	uint32_t others = 0;                    // tokens of the lists of lower blocks
	if (sub > 1) {
		if (t < sub) {
			exchange_send(&s_sum[rank], cta_addr(&s_bar[1]), (uint32_t)t, sum);
			exchange_send(&s_count[rank], cta_addr(&s_bar[1]), (uint32_t)t, late ? kLate : count);
		}
		const bool waited = exchange_wait(cta_addr(&s_bar[1]));
		const bool gave_up = __syncthreads_or(late || !waited) != 0;
		const uint32_t c = s_count[lane & (sub - 1)];
		late = __any_sync(0xffffffffu, c == kLate) || gave_up;
		if (late) {
			if (rank == 0 && t == 0) {
				if (RESIDENT) {
					if (a.status != nullptr) a.status[r] = kInternalWaitTimeout;
				} else {
					atomicCAS(&a.status[r], 0, pack_status(kInternalWaitTimeout, kSiteLogits, w.layer));
				}
			}
			if (gave_up || rank == 0) exchange_leave(cta_addr(&s_bar[0]), 3);
			return;
		}
		sum = 0;
		uint32_t total = 0;
		if (!cuts)
			for (int i = 0; i < sub; ++i) sum += s_sum[i];
		for (int i = 0; i < sub; ++i) {
			if (i < rank) others += s_count[i];
			total += s_count[i];
		}
		if (cuts) {
			for (int i = 0; i < sub; ++i) sum += s_sum[i];
			if (rank == 0) {
				if (t == 0 && total <= (uint32_t)kList) {
					const uint32_t bytes = (total - count) * 8u + (held == 3 ? 8u : 0u);
					asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(cta_addr(&s_bar[2])), "r"(bytes) : "memory");
				}
			} else {
				if (total <= (uint32_t)kList)
					for (uint32_t i = t; i < count; i += kThreads) exchange_send(list + others + i, cta_addr(&s_bar[2]), 0u, list[i]);
				return;      // (nothing is sent to it any more)
			}
		} else {
			mark = share_of(sum, w.draw, 31);
			unsigned long long before = 0;
			for (int i = 0; i < sub; ++i) {
				if (before <= mark && mark < before + s_sum[i]) {
					owner = i;
					break;
				}
				before += s_sum[i];
			}
			if (rank != owner) return;
			mark -= before;
		}
		count = total;
		if (cuts && total <= (uint32_t)kList) {
			late = !exchange_wait(cta_addr(&s_bar[2]));
			if (__syncthreads_or(late)) {
				if (t == 0) {
					if (RESIDENT) {
						if (a.status != nullptr) a.status[r] = kInternalWaitTimeout;
					} else {
						atomicCAS(&a.status[r], 0, pack_status(kInternalWaitTimeout, kSiteLogits, w.layer));
					}
				}
				exchange_leave(cta_addr(&s_bar[0]), 3);
				return;
			}
		}
	} else if (!cuts) {
		mark = share_of(sum, w.draw, 31);
	}
	int token = -2;
	uint32_t weight = 0, number = 0;
	if (none) {
		sum = 0;
	} else if (!cuts) {
		// the 128 tokens that the mark lies in, then the token
		number = count;
		const int steps = (words + 31) / 32 + 2;
		unsigned long long v[4], mine = 0;
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			v[j] = 4 * t + j < steps ? places.sum[4 * t + j] : 0ull;
			mine += v[j];
		}
		unsigned long long upto = mine;
#pragma unroll
		for (int o = 1; o < 32; o *= 2) {
			const unsigned long long z = __shfl_up_sync(0xffffffffu, upto, o);
			if (lane >= o) upto += z;
		}
		if (lane == 31) s_scan[warp] = upto;
		__syncthreads();
		unsigned long long before = upto - mine;
		for (int i = 0; i < warp; ++i) before += s_scan[i];
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			if (before <= mark && mark < before + v[j]) {
				s_select.place = 4 * t + j;
				s_select.target = mark - before;
			}
			before += v[j];
		}
		__syncthreads();
		if (warp != 0) return;
		const int step = (int)s_select.place;
		mark = s_select.target;
		const int v0 = step == 0 ? s0 : (step == steps - 1 ? last : first + 128 * (step - 1)), v1 = step == 0 ? first : (step == steps - 1 ? s1 : min(last, v0 + 128));
		uint32_t g[4];
		unsigned long long own_sum = 0;
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			const int at = v0 + 4 * lane + j;
			const int32_t x = at < v1 ? w.logits[at] : INT32_MIN;
			g[j] = x != INT32_MIN ? weight_of((uint32_t)top - (uint32_t)x, most, w.slope, w.cut) : 0u;
			if (g[j] < floor_w) g[j] = 0u;
			own_sum += g[j];
		}
		upto = own_sum;
#pragma unroll
		for (int o = 1; o < 32; o *= 2) {
			const unsigned long long z = __shfl_up_sync(0xffffffffu, upto, o);
			if (lane >= o) upto += z;
		}
		before = upto - own_sum;
		const uint32_t who = __ballot_sync(0xffffffffu, before <= mark && mark < upto);
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			if (token < 0 && before <= mark && mark < before + g[j]) {
				token = v0 + 4 * lane + j;
				weight = g[j];
			}
			before += g[j];
		}
		token = __shfl_sync(0xffffffffu, token, __ffs(who) - 1);
		weight = __shfl_sync(0xffffffffu, weight, __ffs(who) - 1);
	} else {
		const int n = (int)min(count, (uint32_t)kList);
		const bool complete = reach >= most;      // the list has every token that has a weight
		bool listed = count <= (uint32_t)kList && (complete || w.top_k == 0 || n >= w.top_k);
		// every element: of the list, or of the whole row
		auto each_key = [&](auto f) {
			if (listed) {
				for (int i = t; i < n; i += kThreads) f(list[i]);
			} else {
				const int head = min(V, (4 - mis) & 3), whole = (V - head) >> 2;
				auto one = [&](int32_t x, int v) {
					const uint32_t d = (uint32_t)top - (uint32_t)x;
					if (x != INT32_MIN && d <= most) f((unsigned long long)d << kIndexBits | (uint32_t)v);
				};
				const int4* q = (const int4*)(w.logits + head);
#pragma unroll 1
				for (int k = t; k < whole; k += 4 * kThreads) {
					int4 y[4];
#pragma unroll
					for (int u = 0; u < 4; ++u)
						if (k + u * kThreads < whole) y[u] = __ldcg(q + k + u * kThreads);
#pragma unroll
					for (int u = 0; u < 4; ++u) {
						if (k + u * kThreads >= whole) break;
						const int v = head + 4 * (k + u * kThreads);
						one(y[u].x, v);
						one(y[u].y, v + 1);
						one(y[u].z, v + 2);
						one(y[u].w, v + 3);
					}
				}
				if (t < head) one(w.logits[t], t);
				const int behind = head + 4 * whole + t;
				if (behind < V) one(w.logits[behind], behind);
			}
		};
		auto weight_of_key = [&](unsigned long long key) { return weight_of((uint32_t)(key >> kIndexBits), most, w.slope, w.cut); };
		unsigned long long bound = ~0ull;      // the last key that is kept
		auto added = [&](auto counts) {        // weights (or ones) of the elements that counts() names
			unsigned long long x = 0;
			each_key([&](unsigned long long key) { x += counts(key); });
			return block_sum(x, s_scan);
		};
		const int bits = kIndexBits + 32 - __clz((int)(listed ? far : most));
		if (w.top_k > 0) {
			if (!listed || n > w.top_k) {
				const unsigned long long have = listed ? (unsigned long long)n : added([&](unsigned long long) { return 1ull; });
				if (have > (unsigned long long)w.top_k)
					bound = select_key([&](auto f) { each_key([&](unsigned long long key) { f(key, 1u); }); }, bits, (unsigned long long)w.top_k - 1ull, places, s_select);
			}
			if (w.top_p < (1u << 30)) sum = added([&](unsigned long long key) { return key <= bound ? (unsigned long long)weight_of_key(key) : 0ull; });
		}
		if (w.top_p < (1u << 30)) {
			const unsigned long long enough = share_of(sum, w.top_p, 30);      // (sum is 2^31 at least, so this is 2 at least)
			// the last kept one is the first up to which `enough` lies
			if (w.top_k == 0 && listed && !complete) {
				const unsigned long long have = added([&](unsigned long long key) { return (unsigned long long)weight_of_key(key); });
				listed = have >= enough;
			}
			const int b = kIndexBits + 32 - __clz((int)(listed ? far : most));
			bound = select_key([&](auto f) { each_key([&](unsigned long long key) { if (key <= bound) f(key, weight_of_key(key)); }); }, b, enough - 1ull, places, s_select);
		}
		auto is_kept = [&](unsigned long long key, uint32_t g) { return key <= bound && g >= floor_w; };
		// (sums are below 2^51, counts below 2^20: one word has no room for both, so two sums)
		unsigned long long mass = 0, many = 0;
		each_key([&](unsigned long long key) {
			const uint32_t g = weight_of_key(key);
			if (is_kept(key, g)) {
				mass += g;
				++many;
			}
		});
		sum = block_sum(mass, s_scan);
		number = (uint32_t)block_sum(many, s_scan);
		mark = share_of(sum, w.draw, 31);
		token = (int)select_key(
		    [&](auto f) {
			    each_key([&](unsigned long long key) {
				    const uint32_t g = weight_of_key(key);
				    if (is_kept(key, g)) f(key & (kMostVocab - 1), g);
			    });
		    },
		    kIndexBits, mark, places, s_select);
		if (t == 0) weight = weight_of((uint32_t)top - (uint32_t)w.logits[token], most, w.slope, w.cut);
	}
	if (t != 0) return;
	if (RESIDENT) {
		if (a.out_tokens != nullptr) a.out_tokens[r] = token;
		if (a.out_mass != nullptr) {
			a.out_mass[2 * r] = weight;
			a.out_mass[2 * r + 1] = (int64_t)sum;
		}
		if (a.out_kept != nullptr) a.out_kept[r] = (int32_t)number;
	} else {
		a.best[r] = token < 0 ? 0ull : 1ull << 32 | (0xFFFFFFFFu - (uint32_t)token);
	}
}

void sample_plan(SampleArgs* a) {
	const int sms = sm_count(), most = std::max(1, 2 * sms / a->rows);
	a->shift = 0;
	while (a->shift < 4 && ((a->vocab >> (a->shift + 1) >= 4096 && (2 << a->shift) <= most) || ((a->vocab + (1 << a->shift) - 1) >> a->shift) > kMostSlice - 128)) ++a->shift;
	a->slice = (((a->vocab + (1 << a->shift) - 1) >> a->shift) + 127) & ~127;
	const bool alone = (a->rows << a->shift) <= sms;
	a->keep = SampleSmem::bytes(1, a->slice) + 4096 <= (alone ? (size_t)220 * 1024 : (size_t)0) ? 1 : 0;
}

template <bool RESIDENT, bool KEEP>
cudaError_t sample_launch(SampleArgs a, cudaStream_t st) {
	static PerDeviceOnce once;
	const auto kernel = k_sample<RESIDENT, KEEP>;
	cudaError_t e = once_per_device(once, [&] {
		const cudaError_t x = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
		return x != cudaSuccess ? x : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, KEEP ? 220 * 1024 : (int)SampleSmem::bytes(0, 0));
	});
	if (e != cudaSuccess) return e;
	a.debug_withhold = exchange_debug_take(kExchangeSample);
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3(1u << a.shift, a.rows);
	cfg.blockDim = dim3(kThreads);
	cfg.dynamicSmemBytes = SampleSmem::bytes(KEEP, a.slice);
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

cudaError_t launch_sample(const SampleRow* rows, int m, int vocab, const Scale* scales, unsigned long long* best, int32_t* status, cudaStream_t st) {
	SampleArgs a{};
	a.rows = m; a.vocab = vocab;
	a.desc = rows; a.scales = scales; a.best = best; a.status = status;
	sample_plan(&a);
	return a.keep ? sample_launch<false, true>(a, st) : sample_launch<false, false>(a, st);
}

}  // namespace sslm

using namespace sslm;

extern "C" sslm_status sslm_b200_sample_resident(const sslm_b200_sample* call, void* stream) {
	if (!call || call->struct_size != sizeof(sslm_b200_sample)) return SSLM_INVALID_ARGUMENT;
	const sslm_b200_sample& c = *call;
	if (c.rows < 0 || c.rows > 65535 || c.vocab < 1 || c.vocab > kMostVocab || c.reserved != 0 || c.logits_stride < c.vocab) return SSLM_INVALID_ARGUMENT;
	if (c.rows == 0) return SSLM_OK;
	if (!c.logits || !c.params || !c.draws || (!c.out_tokens && !c.out_mass && !c.out_kept)) return SSLM_INVALID_ARGUMENT;
	for (const void* p : {(const void*)c.logits, (const void*)c.params, (const void*)c.draws, (const void*)c.out_tokens, (const void*)c.out_kept, (const void*)c.row_status})
		if ((uintptr_t)p & 3) return SSLM_MISALIGNED_BUFFER;
	if ((uintptr_t)c.out_mass & 7) return SSLM_MISALIGNED_BUFFER;
	SampleArgs a{};
	a.rows = c.rows; a.vocab = c.vocab;
	a.logits = c.logits; a.logits_stride = c.logits_stride;
	a.params = c.params; a.draws = c.draws;
	a.out_tokens = c.out_tokens; a.out_mass = c.out_mass; a.out_kept = c.out_kept;
	a.status = c.row_status;
	sample_plan(&a);
	if ((a.keep ? sample_launch<true, true>(a, (cudaStream_t)stream) : sample_launch<true, false>(a, (cudaStream_t)stream)) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}
