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
// Two passes over the logits. The first finds the row's maximum and a bound that is likely to lie below what is kept and above nearly all else:
// the least of the maxima of g groups of threads, which leaves about g (ln g + 0.6) tokens above it, and g at least. The second pass lists these tokens,
// a few hundred to two thousand, and adds up the weights where top-p needs that. The list is sorted, cut by its running sums, and what is kept
// sorted by index for the draw. Rows without top-k and top-p need no list: sums of 128 neighbouring tokens are enough to find the token.
//
// Where top-p keeps more than the list has (the sums tell), a sample of the row says where the end of what is kept must lie; a pass adds up
// what is surely kept and lists a window around that end, which is cut as the list is; then the sums of 128 tokens as above. Whatever
// does not work out that way (a list that overflows, a top-k beyond some thousands) is counted into 2,048 places, and those of the place that holds
// the end again, by one block over the whole row.
//
// A row is cut over the blocks of a cluster while rows are few; they exchange maxima and sums, and send their lists to the first one.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

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
// exchanges, in order: maxima and bounds; sums and lists' lengths; the lists; and where the list is too short the window's ends, its sums, its
// lists, the last key that is kept, sums and numbers of what is kept
// (a window's sums take two exchanges in turn, where one window is not enough)
enum { kTop = 0, kSums, kLists, kEnds, kWindow, kWindowLists, kBound, kKept, kWindowOdd, kBars };

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
// d slope / 2^cut with the slope's leading bit moved to bit 30, which changes no quotient: t = hi(d 2^a, m) >> b. `most` is the largest d with a
// weight (t below 2^29), so d 2^a is below 2^31 up to there; it leaves out INT32_MIN too.
struct Scaled {
	uint32_t m, most;
	int a, b;
};
__device__ __forceinline__ Scaled scaled_of(uint32_t slope, uint32_t cut, int32_t top) {
	Scaled s{0u, 0xFFFFFFFFu, 0, 0};
	if (slope != 0u) {
		const int z = __clz((int)slope) - 1, c = (int)cut + z;
		s.m = slope << z;
		s.a = c <= 32 ? min(32 - c, 31) : 0;
		s.b = c <= 32 ? 0 : min(c - 32, 31);
		if (cut < 34u) s.most = (uint32_t)min((unsigned long long)0xFFFFFFFFu, ((1ull << (29 + cut)) - 1ull) / slope);      // (d slope is below 2^63 anyhow)
	}
	s.most = min(s.most, (uint32_t)top - 0x80000001u);
	return s;
}
__device__ __forceinline__ uint32_t weight_of(uint32_t d, const Scaled& s) {
	const uint32_t t = __umulhi(d << s.a, s.m) >> s.b, f = t << 8;
	uint32_t p = 14555373u;
	p = 114090822u - __umulhi(f, p);
	p = 514119776u - __umulhi(f, p);
	p = 1488326151u - __umulhi(f, p);
	p = 2147483648u - __umulhi(f, p);
	p = __funnelshift_rc(p, 0u, t >> 24);
	return d <= s.most ? p : 0u;
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

// ---- the keys of a block in rising order, E of them a thread (thread t those at E t ..), by a bitonic network: partners in the thread, in the warp,
// or by way of `room` (E * kThreads words). The first n of them; those behind are ~0 and stay so.
template <int E>
__device__ __forceinline__ void sort_keys(unsigned long long (&x)[E], int n, unsigned long long* room) {
	const int t = threadIdx.x;
#pragma unroll 1
	for (int k = 2; k < 2 * n; k *= 2) {
#pragma unroll 1
		for (int j = k / 2; j >= E; j /= 2) {
			const int far = j / E;      // threads apart
			const bool up = ((E * t) & k) == 0, low = (t & far) == 0;
			unsigned long long y[E];
			if (far >= 32) {
				__syncthreads();
#pragma unroll
				for (int e = 0; e < E; ++e) room[e * kThreads + t] = x[e];
				__syncthreads();
#pragma unroll
				for (int e = 0; e < E; ++e) y[e] = room[e * kThreads + (t ^ far)];
			} else {
#pragma unroll
				for (int e = 0; e < E; ++e) y[e] = __shfl_xor_sync(0xffffffffu, x[e], far);
			}
#pragma unroll
			for (int e = 0; e < E; ++e) x[e] = (low == up) == (x[e] < y[e]) ? x[e] : y[e];
		}
#pragma unroll
		for (int j = E / 2; j > 0; j /= 2) {
			if (j >= k) continue;
#pragma unroll
			for (int e = 0; e < E; ++e) {
				if ((e & j) != 0) continue;
				const bool up = ((E * t + e) & k) == 0;
				const unsigned long long a = x[e], b = x[e | j];
				x[e] = (a < b) == up ? a : b;
				x[e | j] = (a < b) == up ? b : a;
			}
		}
	}
}
// sums of v over the elements in front of each of a thread's own, in that order
template <int E>
__device__ __forceinline__ void sums_before(const uint32_t (&v)[E], unsigned long long (&before)[E], unsigned long long* s) {
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	unsigned long long mine = 0;
#pragma unroll
	for (int e = 0; e < E; ++e) mine += v[e];
	unsigned long long upto = mine;
#pragma unroll
	for (int o = 1; o < 32; o *= 2) {
		const unsigned long long z = __shfl_up_sync(0xffffffffu, upto, o);
		if (lane >= o) upto += z;
	}
	__syncthreads();
	if (lane == 31) s[warp] = upto;
	__syncthreads();
	unsigned long long at = upto - mine;
	for (int i = 0; i < warp; ++i) at += s[i];
#pragma unroll
	for (int e = 0; e < E; ++e) {
		before[e] = at;
		at += v[e];
	}
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

// What a list of a row is cut by, and what came of it.
struct Cut {
	Scaled scale;
	unsigned long long origin;   // of the list's keys: they are (INT32_MAX - x) 2^20 + v, and less it d 2^20 + v
	uint32_t floor_w, top_p, draw;
	int top_k;
	unsigned long long sum;      // of all weights, where top-k does not say what counts
};
struct Drawn {
	int token;
	uint32_t weight, number;
	unsigned long long sum;
};
__device__ __forceinline__ uint32_t key_weight(unsigned long long key, const Cut& c) { return weight_of((uint32_t)(key >> kIndexBits), c.scale); }

// The list in the order of falling logits, cut, and drawn from. n <= E * kThreads keys, which are overwritten. For the threads of a whole block.
template <int E>
__device__ __noinline__ Drawn draw_sorted(unsigned long long* list, int n, const Cut& c, unsigned long long* s_scan, Drawn* s_drawn) {
	const int t = threadIdx.x, lane = t & 31;
	unsigned long long x[E], before[E];
	uint32_t w[E];
#pragma unroll
	for (int e = 0; e < E; ++e) x[e] = E * t + e < n ? list[E * t + e] - c.origin : ~0ull;
	__syncthreads();
	sort_keys<E>(x, n, list);
	unsigned long long sum = 0;
	const int limit = c.top_k > 0 ? min(n, c.top_k) : n;
#pragma unroll
	for (int e = 0; e < E; ++e) {
		w[e] = E * t + e < limit ? key_weight(x[e], c) : 0u;
		sum += w[e];
	}
	sum = c.top_k > 0 ? block_sum(sum, s_scan) : c.sum;
	const unsigned long long enough = c.top_p < (1u << 30) ? share_of(sum, c.top_p, 30) : ~0ull;
	sums_before<E>(w, before, s_scan);
	unsigned long long mass = 0;
	uint32_t many = 0;
#pragma unroll
	for (int e = 0; e < E; ++e) {
		const bool yes = before[e] < enough && w[e] >= c.floor_w;
		if (!yes) w[e] = 0u;
		mass += w[e];
		many += yes ? 1u : 0u;
	}
	mass = block_sum(mass, s_scan);
	const int kept = (int)block_sum(many, s_scan);      // (the first so many)
	const unsigned long long mark = share_of(mass, c.draw, 31);
	// by index
	if (kept <= 32) {
#pragma unroll
		for (int e = 0; e < E; ++e)
			if (E * t + e < kept) list[E * t + e] = (x[e] & (kMostVocab - 1)) << 32 | w[e];
		__syncthreads();
		if (t < 32) {
			const unsigned long long mine = lane < kept ? list[lane] : ~0ull;
			unsigned long long less = 0;
			for (int i = 0; i < kept; ++i) {
				const unsigned long long y = list[i];
				if (y < mine) less += (uint32_t)y;
			}
			if (lane < kept && less <= mark && mark < less + (uint32_t)mine) *s_drawn = Drawn{(int)(mine >> 32), (uint32_t)mine, (uint32_t)kept, mass};
		}
	} else {
#pragma unroll
		for (int e = 0; e < E; ++e) x[e] = E * t + e < kept ? (x[e] & (kMostVocab - 1)) << 32 | w[e] : ~0ull;
		sort_keys<E>(x, kept, list);
#pragma unroll
		for (int e = 0; e < E; ++e) w[e] = E * t + e < kept ? (uint32_t)x[e] : 0u;
		sums_before<E>(w, before, s_scan);
#pragma unroll
		for (int e = 0; e < E; ++e)
			if (before[e] <= mark && mark < before[e] + w[e]) *s_drawn = Drawn{(int)(x[e] >> 32), w[e], (uint32_t)kept, mass};
	}
	__syncthreads();
	return *s_drawn;
}

template <bool RESIDENT, bool KEEP>
__global__ void __launch_bounds__(kThreads, KEEP ? 1 : 2) k_sample(const __grid_constant__ SampleArgs a) {
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ __align__(8) unsigned long long s_bar[kBars], s_sum[3][16], s_scan[kWarps], s_bound;
	__shared__ int2 s_top[16], s_warp[kWarps], s_ends;
	__shared__ uint32_t s_count[3][16], s_n;
	__shared__ Row s_row;
	__shared__ Drawn s_drawn;
	__shared__ unsigned long long s_listed[3][16];
	__shared__ SelectSmem s_select;
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.vocab;
	const int sub = 1 << a.shift, rank = (int)blockIdx.x;
	const int64_t r = blockIdx.y;
	unsigned long long* list = (unsigned long long*)smem;
	const Place places{list + kList, (uint32_t*)(list + kList + kPlaces)};
	int4* kept = (int4*)(places.count + kPlaces);
	// 1 + the exchange that is made to run out, in the first block, or where the first one only sends, in the second
	const bool sends = a.debug_withhold == 1 + kEnds || a.debug_withhold == 1 + kBound;
	const int held = blockIdx.y == 0 && rank == (sends ? 1 : 0) ? a.debug_withhold : 0;
	if (t == 0) {
		if (sub > 1) {
			exchange_init(cta_addr(&s_bar[kTop]), (uint32_t)(sub * 8) + (held == 1 + kTop ? 4u : 0u));
			exchange_init(cta_addr(&s_bar[kSums]), (uint32_t)(sub * 20) + (held == 1 + kSums ? 4u : 0u));
			ring_init(cta_addr(&s_bar[kLists]), 1);      // (armed when the lists' lengths are known)
			exchange_init(cta_addr(&s_bar[kEnds]), 8u + (held == 1 + kEnds ? 4u : 0u));
			exchange_init(cta_addr(&s_bar[kWindow]), (uint32_t)(sub * 20) + (held == 1 + kWindow ? 4u : 0u));
			ring_init(cta_addr(&s_bar[kWindowLists]), 1);
			exchange_init(cta_addr(&s_bar[kBound]), 8u + (held == 1 + kBound ? 4u : 0u));
			exchange_init(cta_addr(&s_bar[kWindowOdd]), (uint32_t)(sub * 20));
			exchange_init(cta_addr(&s_bar[kKept]), (uint32_t)(sub * 12) + (held == 1 + kKept ? 4u : 0u));
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
	constexpr int U = 4;
	const int rounds = (words + U * kThreads - 1) / (U * kThreads);      // of U words a thread
	// f(the word, its first token, its number), over the block's words, the next ones asked for ahead; LAST: from the last ones on (what was read last is
	// likelier still in L2). Words behind the last are INT32_MIN where ALL threads of a warp are to take part.
	auto each_word = [&](auto last_first, auto all, auto stored, auto f) {
		constexpr bool LAST = decltype(last_first)::value, ALL = decltype(all)::value, STORED = decltype(stored)::value;
		int4 q[U], y[U];
		auto fetch = [&](int4 (&to)[U], int i) {
			const int k = (LAST ? rounds - 1 - i : i) * U * kThreads + t;
#pragma unroll
			for (int u = 0; u < U; ++u)
				if (k + u * kThreads < words) to[u] = STORED ? kept[k + u * kThreads] : __ldcg(from + k + u * kThreads);
		};
		if (rounds > 0) fetch(q, 0);
#pragma unroll 1
		for (int i = 0; i < rounds; ++i) {
			if (i + 1 < rounds) fetch(y, i + 1);
			const int k = (LAST ? rounds - 1 - i : i) * U * kThreads + t;
#pragma unroll
			for (int u = 0; u < U; ++u) {
				const bool there = k + u * kThreads < words;
				if (ALL && !there) q[u] = make_int4(INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN);
				if (ALL || there) f(q[u], first + 4 * (k + u * kThreads), k + u * kThreads);
				q[u] = y[u];
			}
		}
	};
	using Yes = std::true_type;
	using No = std::false_type;
	using Kept = std::integral_constant<bool, KEEP>;
	auto put = [&](int32_t x, int v) {
		const uint32_t at = atomicAdd(&s_n, 1u);
		if (at < (uint32_t)kList) list[at] = (unsigned long long)(0x7FFFFFFFu - (uint32_t)x) << kIndexBits | (uint32_t)v;
	};
	auto put_from = [&](int4 q, int v, int32_t least) {      // the tokens of a word from `least` on
		if (max(max(q.x, q.y), max(q.z, q.w)) < least) return;
		if (q.x >= least) put(q.x, v);
		if (q.y >= least) put(q.y, v + 1);
		if (q.z >= least) put(q.z, v + 2);
		if (q.w >= least) put(q.w, v + 3);
	};
	// a wait ran out: the row is reported, and the block stays until nothing can be sent to it any more
	auto give_up = [&](bool stay) {
		if (t == 0) {
			if (RESIDENT) {
				if (a.status != nullptr) a.status[r] = kInternalWaitTimeout;
			} else {
				atomicCAS(&a.status[r], 0, pack_status(kInternalWaitTimeout, kSiteLogits, w.layer));
			}
		}
		if (stay) exchange_leave(cta_addr(&s_bar[0]), kBars);
	};

	// ---- the maximum, and the least of the groups' maxima
	int32_t top = end_x;
	// One block has a long row and a small top-k: the least of the maxima of the row's first eighth, of 16 to 64 groups, leaves eight times as
	// many tokens of the row as of that eighth, so the list can be made in the first pass already (256 rows: a pass less).
	const bool early = !KEEP && sub == 1 && w.top_k > 0 && w.top_k <= 400 && words >= 16 * kThreads;
	int32_t early_least = INT32_MIN;
	if (early) {
		int32_t m = INT32_MIN;
		const int part = words / (8 * kThreads) * kThreads;
#pragma unroll 4
		for (int k = t; k < part; k += kThreads) {
			const int4 q = __ldcg(from + k);
			m = max(m, max(max(q.x, q.y), max(q.z, q.w)));
		}
		const int mates = w.top_k <= 64 ? 32 : (w.top_k <= 160 ? 16 : 8);      // threads of a group
		for (int o = 1; o < mates; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
		m = __reduce_min_sync(0xffffffffu, m);
		if (lane == 0) s_warp[warp] = make_int2(m, 0);
		__syncthreads();
		early_least = max(INT32_MIN + 1, __reduce_min_sync(0xffffffffu, s_warp[lane & (kWarps - 1)].x));
		if (end_x >= early_least) put(end_x, end);
		each_word(No(), No(), No(), [&](int4 q, int v, int) {
			top = max(top, max(max(q.x, q.y), max(q.z, q.w)));
			put_from(q, v, early_least);
		});
		__syncthreads();      // (s_warp is used again)
	} else {
		each_word(No(), No(), No(), [&](int4 q, int, int k) {
			if (KEEP) kept[k] = q;
			top = max(top, max(max(q.x, q.y), max(q.z, q.w)));
		});
	}
	const bool cuts = w.top_k > 0 || w.top_p < (1u << 30);
	int32_t least = INT32_MAX;
	int group = 1;      // threads of a group, over all blocks 256 groups, or as many as there are tokens to keep
	if (cuts) {
		int wanted = 256;
		if (w.top_k > 0) {
			wanted = 32;
			while (wanted < min(w.top_k, 512)) wanted *= 2;
		}
		group = max(1, min(kThreads, sub * kThreads / wanted));
		const bool has = t < words || end >= 0;
		least = has ? top : INT32_MIN;
		for (int o = 1; o < min(group, 32); o *= 2) least = max(least, __shfl_xor_sync(0xffffffffu, least, o));
		// (threads without a token count only where their whole group has none)
		const uint32_t any = __ballot_sync(0xffffffffu, has);
		const uint32_t mates = group >= 32 ? 0xFFFFFFFFu : ((1u << group) - 1u) << (lane & ~(group - 1));
		if ((any & mates) == 0u) least = INT32_MAX;
	}
	{
		const int32_t m = __reduce_max_sync(0xffffffffu, top), l = __reduce_min_sync(0xffffffffu, least);
		if (lane == 0) s_warp[warp] = make_int2(m, l);
	}
	__syncthreads();
	{
		const int2 x = s_warp[lane & (kWarps - 1)];
		top = __reduce_max_sync(0xffffffffu, x.x);
		least = x.y;
		for (int o = 1; o < group / 32; o *= 2) {
			const int32_t y = __shfl_xor_sync(0xffffffffu, least, o);
			least = least == INT32_MAX ? y : (y == INT32_MAX ? least : max(least, y));
		}
		least = __reduce_min_sync(0xffffffffu, least);
		if (top == INT32_MIN) least = INT32_MAX;      // (nothing is allowed here)
	}
	bool late = false;
	if (sub > 1) {
		cluster_wait();      // (all blocks run)
		if (t < sub) exchange_send(&s_top[rank], cta_addr(&s_bar[kTop]), (uint32_t)t, make_int2(top, least));
		late = !exchange_wait(cta_addr(&s_bar[kTop]));
		const int2 x = s_top[lane & (sub - 1)];
		top = __reduce_max_sync(0xffffffffu, x.x);
		least = __reduce_min_sync(0xffffffffu, x.y);
		late = __syncthreads_or(late) != 0;
	}
	const bool none = top == INT32_MIN;
	const Scaled scale = scaled_of(w.slope, w.cut, none ? INT32_MAX : top);
	const uint32_t most = scale.most, floor_w = max(1u, 2u * w.min_p);
	auto weight = [&](int32_t x) { return weight_of((uint32_t)top - (uint32_t)x, scale); };
	// sums over all tokens that counts() names, of 128 neighbours each: places 1 .. , the ends at 0 and behind
	unsigned long long sum = 0, listed = 0;
	uint32_t count = 0;
	const int steps = (words + 31) / 32 + 2;
	auto add_steps = [&](auto counts) {
		if (t < 2) places.sum[t == 0 ? 0 : steps - 1] = 0ull;
		__syncthreads();
		if (end >= 0) {
			const uint32_t g = counts(end_x, end);
			sum += g;
			count += g != 0u ? 1u : 0u;
			atomicAdd(&places.sum[t < 4 ? 0 : steps - 1], (unsigned long long)g);
		}
		each_word(Yes(), Yes(), Kept(), [&](int4 q, int v, int k) {
			const uint32_t g0 = counts(q.x, v), g1 = counts(q.y, v + 1), g2 = counts(q.z, v + 2), g3 = counts(q.w, v + 3);
			const unsigned long long g = (unsigned long long)g0 + g1 + g2 + g3;
			sum += g;
			count += (g0 != 0u ? 1u : 0u) + (g1 != 0u ? 1u : 0u) + (g2 != 0u ? 1u : 0u) + (g3 != 0u ? 1u : 0u);
			const uint32_t high = __reduce_add_sync(0xffffffffu, (uint32_t)(g >> 16)), low = __reduce_add_sync(0xffffffffu, (uint32_t)g & 0xFFFFu);
			if (lane == 0 && k < words) places.sum[1 + (k >> 5)] = ((unsigned long long)high << 16) + low;
		});
	};

	// ---- the second pass
	const uint32_t reach = least == INT32_MIN ? 0xFFFFFFFFu : (uint32_t)top - (uint32_t)max(least, INT32_MIN + 1), far = min(reach, most);      // the list's farthest
	bool complete = reach >= most;      // the list has every token that has a weight
	const bool have_list = early && s_n >= (uint32_t)w.top_k && s_n <= (uint32_t)kList;
	if (early) {
		__syncthreads();      // (all have seen how long it is)
		if (have_list) complete = false;
		else if (t == 0) s_n = 0u;
		__syncthreads();
	}
	if (!late && !none && !have_list) {
		if (!cuts) {
			add_steps([&](int32_t x, int) {
				const uint32_t g = weight(x);
				return g >= floor_w ? g : 0u;
			});
		} else {
			const int32_t from_x = (int32_t)max((long long)top - (long long)far, -2147483647ll);
			if (w.top_k == 0) {      // all weights are added up, and those of the list
				auto one = [&](int32_t x, int v) {
					const uint32_t g = weight(x);
					sum += g;
					if (x >= from_x) {
						listed += g;
						put(x, v);
					}
				};
				one(end_x, end);
				each_word(Yes(), No(), Kept(), [&](int4 q, int v, int) {
					one(q.x, v);
					one(q.y, v + 1);
					one(q.z, v + 2);
					one(q.w, v + 3);
				});
			} else {
				if (end_x >= from_x) put(end_x, end);
				each_word(Yes(), No(), Kept(), [&](int4 q, int v, int) { put_from(q, v, from_x); });
			}
		}
	}
	sum = block_sum(sum, s_scan);      // (a barrier, behind which the list is whole)
	if (!cuts) {
		count = (uint32_t)block_sum(count, s_scan);
	} else {
		if (w.top_k == 0) listed = block_sum(listed, s_scan);
		count = s_n;
	}
	int owner = 0;                          // the block that finds the token among its sums
	unsigned long long mark = 0;            // what it looks for
	// sums of all blocks: of `what` words; false where a wait ran out here or elsewhere
	auto tell = [&](int bar, int slot, bool both, uint32_t turn) {
		if (t < sub) {
			exchange_send(&s_sum[slot][rank], cta_addr(&s_bar[bar]), (uint32_t)t, sum);
			if (both) exchange_send(&s_listed[slot][rank], cta_addr(&s_bar[bar]), (uint32_t)t, listed);
			exchange_send(&s_count[slot][rank], cta_addr(&s_bar[bar]), (uint32_t)t, late ? kLate : count);
		}
		const bool waited = bounded_wait<true>(cta_addr(&s_bar[bar]), turn & 1u);
		const bool gave_up = __syncthreads_or(late || !waited) != 0;
		const uint32_t c = s_count[slot][lane & (sub - 1)];
		if (!__any_sync(0xffffffffu, c == kLate) && !gave_up) return true;
		give_up(gave_up || rank == 0);
		return false;
	};
	// of a total that all blocks have, what lies before the mark in other blocks
	auto find_owner = [&](int slot) {
		unsigned long long before = 0;
		owner = 0;
		for (int i = 0; i < sub; ++i) {
			if (before <= mark && mark < before + s_sum[slot][i]) {
				owner = i;
				break;
			}
			before += s_sum[slot][i];
		}
		mark -= rank == owner ? before : 0ull;
	};
	uint32_t others = 0;                    // tokens of the lists of lower blocks
	uint32_t total = count;
	if (sub > 1) {
		if (!tell(kSums, 0, true, 0u)) return;
		sum = listed = 0;
		total = 0;
		for (int i = 0; i < sub; ++i) {
			sum += s_sum[0][i];
			listed += s_listed[0][i];
			if (i < rank) others += s_count[0][i];
			total += s_count[0][i];
		}
	}
	Drawn out{-2, 0u, 0u, 0ull};
	bool by_steps = !cuts;
	if (cuts && !none) {
		const Cut cut{scale, (unsigned long long)(0x7FFFFFFFu - (uint32_t)top) << kIndexBits, floor_w, w.top_p, w.draw, w.top_k, sum};
		const unsigned long long enough = w.top_k == 0 ? share_of(sum, w.top_p, 30) : 0ull;
		bool wide = false;
		unsigned long long bound = ~0ull, sure = 0;      // the last key that is kept; weights in front of the window
		unsigned long long kept_sum = 0;                 // this block's kept ones in front of the window
		uint32_t kept_count = 0;
		const bool fits = total <= (uint32_t)kList && (complete || (w.top_k > 0 ? total >= (uint32_t)w.top_k : listed >= enough));
		if (!fits) {
			wide = w.top_k == 0 && total <= (uint32_t)kList;
			// what is kept ends at a d in (begin, stop], up to which exactly `before` and `through` of the weights lie
			uint32_t begin = far, stop = most, turn = 0;
			unsigned long long before_begin = listed, through_stop = sum;
			while (wide) {
				// ---- a sample (32,768 to 65,536 of the first block's tokens, or all) says where in between, to one or two in a hundred; the window
				// is three to either side, or less where that would be too many tokens
				if (rank == 0) {
					const int down = max(0, 32 - __clz((int)(stop - begin)) - 11);
					for (int i = t; i < kPlaces; i += kThreads) places.count[i] = 0u;
					__syncthreads();
					const int every = max(1, words / 8192);
					for (int k = t * every; k < words; k += kThreads * every) {
						const int4 q = KEEP ? kept[k] : __ldcg(from + k);
						const int32_t y[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
						for (int j = 0; j < 4; ++j) {
							const uint32_t d = (uint32_t)top - (uint32_t)y[j];
							if (d > begin && d <= stop) atomicAdd(&places.count[min((d - begin - 1u) >> down, (uint32_t)kPlaces - 1u)], 1u);
						}
					}
					__syncthreads();
					// weights of the places, in units such that none is above 2^15 (and no place's sum above 2^31)
					const int shift = max(0, 17 - __clz((int)weight_of(begin, scale)));
					uint32_t v[4];
					unsigned long long at[4], all = 0;
#pragma unroll
					for (int j = 0; j < 4; ++j) {
						const uint32_t i = 4 * t + j, mid = begin + 1u + (i << down) + ((1u << down) >> 1);
						v[j] = mid > begin ? places.count[i] * (weight_of(mid, scale) >> shift) : 0u;
						all += v[j];
					}
					all = block_sum(all, s_scan);
					sums_before<4>(v, at, s_scan);
					const double want = (double)(enough - before_begin) / (double)(through_stop - before_begin);
					double slack = 0.03;
					unsigned long long number[2];      // of the sample, in the window
					for (int turn_of = 0; turn_of < 2; ++turn_of) {
						const double low = (want - slack) * (double)all, high = (want + slack) * (double)all;
						if (t == 0) s_ends = make_int2((int)begin, (int)stop);
						__syncthreads();
						uint32_t in = 0;
#pragma unroll
						for (int j = 0; j < 4; ++j) {
							const uint32_t i = 4 * t + j;
							if ((double)at[j] <= low && low < (double)(at[j] + v[j])) s_ends.x = (int)(begin + (i << down));
							if ((double)at[j] <= high && high < (double)(at[j] + v[j]))
								s_ends.y = (int)min((unsigned long long)stop, (unsigned long long)begin + ((unsigned long long)(i + 1) << down));
							if ((double)(at[j] + v[j]) > low && (double)at[j] <= high) in += places.count[i];
						}
						number[turn_of] = block_sum(in, s_scan) * (unsigned long long)(every * sub);
						if (number[turn_of] <= (unsigned long long)kList * 3 / 4) break;
						slack = max(0.01, slack * (double)(kList / 2) / (double)number[turn_of]);
						__syncthreads();
					}
					__syncthreads();
					if (sub > 1 && t < sub && t != 0) exchange_send(&s_ends, cta_addr(&s_bar[kEnds]), (uint32_t)t, s_ends);
				} else {
					late = !bounded_wait<true>(cta_addr(&s_bar[kEnds]), turn & 1u);
					if (__syncthreads_or(late)) {
						give_up(true);
						return;
					}
				}
				const uint32_t near = (uint32_t)s_ends.x, until = (uint32_t)s_ends.y;      // the window: near < d <= until
				__syncthreads();
				if (t == 0) s_n = 0u;
				// ---- a pass: weights up to the window, and of what is kept of them by 128 tokens; weights and list of the window
				sum = listed = 0;
				count = 0;
				kept_sum = 0;
				const int32_t until_x = (int32_t)max((long long)top - (long long)until, -2147483647ll), near_x = (int32_t)max((long long)top - (long long)near, -2147483647ll);
				add_steps([&](int32_t x, int v) {
					uint32_t g = 0;
					if (x >= until_x) {
						g = weight(x);
						if (x >= near_x) {
							kept_sum += g;
							g = g >= floor_w ? g : 0u;
						} else {
							listed += g;
							put(x, v);
							g = 0u;
						}
					}
					return g;
				});
				const unsigned long long own_sum = sum;
				kept_count = count;
				sum = block_sum(kept_sum, s_scan);      // (of all weights up to the window)
				listed = block_sum(listed, s_scan);
				kept_sum = block_sum(own_sum, s_scan);
				kept_count = (uint32_t)block_sum(kept_count, s_scan);
				count = total = s_n;
				others = 0;
				if (sub > 1) {
					const int slot = 1 + (int)(turn & 1u);
					if (!tell(slot == 1 ? kWindow : kWindowOdd, slot, true, turn >> 1)) return;
					sum = listed = 0;
					total = 0;
					for (int i = 0; i < sub; ++i) {
						sum += s_sum[slot][i];
						listed += s_listed[slot][i];
						if (i < rank) others += s_count[slot][i];
						total += s_count[slot][i];
					}
				}
				sure = sum;
				if (sure < enough && enough <= sure + listed && total <= (uint32_t)kList) break;      // (the last kept one is the first up to which `enough` lies)
				// not in the window, or more tokens than the list holds: closer in, for a few turns
				if (enough <= sure) {
					stop = near;
					through_stop = sure;
				} else if (enough <= sure + listed) {
					begin = near;
					before_begin = sure;
					stop = until;
					through_stop = sure + listed;
				} else {
					begin = until;
					before_begin = sure + listed;
				}
				wide = ++turn < 6u && stop - begin > 1u;
				if (sub > 1 && wide) {
					if (t == 0) {      // (of the next turn's ends and the next but one's sums; what comes may have come already)
						asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(cta_addr(&s_bar[(turn & 1u) != 0u ? kWindow : kWindowOdd])), "r"((uint32_t)(sub * 20)) : "memory");
						if (rank != 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(cta_addr(&s_bar[kEnds])), "r"(8u) : "memory");
					}
					__syncthreads();
				}
			}
			if (!wide && rank != 0) return;
		}
		const bool do_list = wide || fits;
		const uint32_t own_listed = count;      // (at the front of the list)
		if (sub > 1 && do_list) {      // the lists, to the first block
			const uint32_t bar = cta_addr(&s_bar[wide ? kWindowLists : kLists]);
			if (rank != 0) {
				for (uint32_t i = t; i < count; i += kThreads) exchange_send(list + others + i, bar, 0u, list[i]);
				if (!wide) return;      // (nothing is sent to it any more)
			} else {
				if (t == 0) {
					const uint32_t bytes = (total - count) * 8u + (held == 1 + (wide ? kWindowLists : kLists) ? 8u : 0u);
					asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
				}
				late = !exchange_wait(bar);
				if (__syncthreads_or(late)) {
					give_up(true);
					return;
				}
			}
		}
		if (wide) {
			if (rank == 0) {
				unsigned long long aside[4];      // (the sums of 128 tokens: the selection needs their places)
#pragma unroll
				for (int j = 0; j < 4; ++j) aside[j] = places.sum[4 * t + j];
				__syncthreads();
				bound = select_key(
				    [&](auto f) {
					    for (int i = t; i < (int)total; i += kThreads) f(list[i] - cut.origin, key_weight(list[i] - cut.origin, cut));
				    },
				    kIndexBits + 32 - __clz((int)most), enough - 1ull - sure, places, s_select);
#pragma unroll
				for (int j = 0; j < 4; ++j) places.sum[4 * t + j] = aside[j];
				if (t == 0) s_bound = bound;
				__syncthreads();
				if (sub > 1 && t < sub && t != 0) exchange_send(&s_bound, cta_addr(&s_bar[kBound]), (uint32_t)t, bound);
			} else {
				late = !exchange_wait(cta_addr(&s_bar[kBound]));
				if (__syncthreads_or(late)) {
					give_up(true);
					return;
				}
				bound = s_bound;
			}
			// the block's tokens of the window that are kept, to their 128 neighbours
			sum = 0;
			count = 0;
			for (uint32_t i = t; i < own_listed; i += kThreads) {
				const unsigned long long key = list[i] - cut.origin;
				const uint32_t g = key_weight(key, cut);
				if (key > bound || g < floor_w) continue;
				const int v = (int)(key & (kMostVocab - 1));
				sum += g;
				++count;
				atomicAdd(&places.sum[v < first ? 0 : (v >= last ? steps - 1 : 1 + ((v - first) >> 7))], (unsigned long long)g);
			}
			sum = block_sum(sum, s_scan) + kept_sum;
			count = total = (uint32_t)block_sum(count, s_scan) + kept_count;
			if (sub > 1) {
				if (!tell(kKept, 0, false, 0u)) return;
				sum = 0;
				total = 0;
				for (int i = 0; i < sub; ++i) {
					sum += s_sum[0][i];
					total += s_count[0][i];
				}
			}
			by_steps = true;
		} else if (do_list && total <= 8u * kThreads) {
			out = total <= (uint32_t)kThreads ? draw_sorted<1>(list, (int)total, cut, s_scan, &s_drawn)
			                                  : (total <= 4u * kThreads ? draw_sorted<4>(list, (int)total, cut, s_scan, &s_drawn) : draw_sorted<8>(list, (int)total, cut, s_scan, &s_drawn));
		} else {
			// every element: of the list, or of the whole row
			auto each_key = [&](auto f) {
				if (do_list) {
					for (int i = t; i < (int)total; i += kThreads) f(list[i] - cut.origin);
				} else {
					const int head = min(V, (4 - mis) & 3), whole = (V - head) >> 2;
					auto one = [&](int32_t x, int v) {
						const uint32_t d = (uint32_t)top - (uint32_t)x;
						if (d <= most) f((unsigned long long)d << kIndexBits | (uint32_t)v);
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
			auto added = [&](auto counts) {        // weights (or ones) of the elements that counts() names
				unsigned long long x = 0;
				each_key([&](unsigned long long key) { x += counts(key); });
				return block_sum(x, s_scan);
			};
			const int bits = kIndexBits + 32 - __clz((int)most);
			if (w.top_k > 0) {
				if (added([&](unsigned long long) { return 1ull; }) > (unsigned long long)w.top_k)
					bound = select_key([&](auto f) { each_key([&](unsigned long long key) { f(key, 1u); }); }, bits, (unsigned long long)w.top_k - 1ull, places, s_select);
				if (w.top_p < (1u << 30)) sum = added([&](unsigned long long key) { return key <= bound ? (unsigned long long)key_weight(key, cut) : 0ull; });
			} else {
				sum = cut.sum;
			}
			if (w.top_p < (1u << 30))
				bound = select_key([&](auto f) { each_key([&](unsigned long long key) { if (key <= bound) f(key, key_weight(key, cut)); }); }, bits, share_of(sum, w.top_p, 30) - 1ull,
				                   places, s_select);
			auto is_kept = [&](unsigned long long key, uint32_t g) { return key <= bound && g >= floor_w; };
			unsigned long long mass = 0, many = 0;
			each_key([&](unsigned long long key) {
				const uint32_t g = key_weight(key, cut);
				if (is_kept(key, g)) {
					mass += g;
					++many;
				}
			});
			out.sum = block_sum(mass, s_scan);
			out.number = (uint32_t)block_sum(many, s_scan);
			out.token = (int)select_key(
			    [&](auto f) {
				    each_key([&](unsigned long long key) {
					    const uint32_t g = key_weight(key, cut);
					    if (is_kept(key, g)) f(key & (kMostVocab - 1), g);
				    });
			    },
			    kIndexBits, share_of(out.sum, w.draw, 31), places, s_select);
			if (t == 0) out.weight = weight(w.logits[out.token]);
		}
	}
	if (by_steps && !none) {
		// the 128 tokens that the mark lies in, then the token
		mark = share_of(sum, w.draw, 31);
		if (sub > 1) find_owner(0);
		if (rank != owner) return;
		out.sum = sum;
		out.number = total;
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
		const unsigned long long bound = cuts ? s_bound : ~0ull;
		const int v0 = step == 0 ? s0 : (step == steps - 1 ? last : first + 128 * (step - 1)), v1 = step == 0 ? first : (step == steps - 1 ? s1 : min(last, v0 + 128));
		uint32_t g[4];
		unsigned long long own_sum = 0;
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			const int at = v0 + 4 * lane + j;
			const int32_t x = at < v1 ? w.logits[at] : INT32_MIN;
			g[j] = weight(x);      // (none of INT32_MIN)
			if (g[j] < floor_w || ((unsigned long long)((uint32_t)top - (uint32_t)x) << kIndexBits | (uint32_t)at) > bound) g[j] = 0u;
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
			if (out.token < 0 && before <= mark && mark < before + g[j]) {
				out.token = v0 + 4 * lane + j;
				out.weight = g[j];
			}
			before += g[j];
		}
		out.token = __shfl_sync(0xffffffffu, out.token, __ffs(who) - 1);
		out.weight = __shfl_sync(0xffffffffu, out.weight, __ffs(who) - 1);
	} else if (rank != 0) {
		return;
	}
	if (t != 0) return;
	if (RESIDENT) {
		if (a.out_tokens != nullptr) a.out_tokens[r] = out.token;
		if (a.out_mass != nullptr) {
			a.out_mass[2 * r] = out.weight;
			a.out_mass[2 * r + 1] = (int64_t)out.sum;
		}
		if (a.out_kept != nullptr) a.out_kept[r] = (int32_t)out.number;
	} else {
		a.best[r] = out.token < 0 ? 0ull : 1ull << 32 | (0xFFFFFFFFu - (uint32_t)out.token);
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
