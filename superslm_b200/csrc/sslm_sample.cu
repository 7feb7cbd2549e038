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
// a few hundred to two thousand, and adds up the weights where top-p needs that. The list is cut and drawn from by counting its weights into 512
// places. Rows without top-k and top-p need no list: sums of 256 neighbouring tokens are enough to find the token.
//
// Where top-p keeps more than the list has (the sums tell), a sample of the row says where the end of what is kept must lie; a pass adds up
// what is surely kept and lists a window around that end, which is cut as the list is; then the sums of 256 tokens as above. Whatever
// does not work out that way is counted by one block over the whole row, in some 20 passes: a list that overflows, or one with fewer tokens
// than top-k. The groups are 512 at most, and the least of 512 maxima leaves 3,440 tokens on the average (of normal logits; 2,500 to 4,900
// in 60 rows), so that is where a large top-k ends up: in some rows from 2,500 on, in nearly all above 4,500. Rows of 151,936, us: 64 rows with top-k
// 2,000 41, 2,500 286, 4,000 399; one row 22, 22, 361.
//
// A row is cut over the blocks of a cluster while rows are few; they exchange maxima and sums, and send their lists to the first one.
//
// Rows of 151,936 logits, us: one row with top-k 50 and top-p 10.0, 21 rows with a temperature alone 13.2, 64 with top-p 0.9 of which 2,400 tokens are kept on
// the average 79, 256 with top-k 40 and top-p 44.5; 40 rows of 32,003 of which a schema allows 1,000, top-p, 16.3. What bounds them, by a block's clock
// (cycles at 1.9 GHz):
//   one row    its chain: the maximum 2,900, the list 3,900, their exchanges 900 and 2,400, the lists' exchange, cut and draw 7,800
//   21 rows    the second pass with 12,100 of 23,700 (a pass of weights keeps a scheduler busy for 49 cycles a warp's 32 tokens, one that lists besides 60 to
//              85), then the first pass 3,000, exchanges 2,000 and 2,400, the search of the token 3,000
//   40 rows    the lists' exchange and the selections in one block with 13,200 of 28,400, then the second pass with 8,000, which weighs masked tokens too
//   64 rows    their passes, the window's among them, which weighs every token though few count there (45 % of the issue slots are used)
//   256 rows   the first pass, 57,000 of 76,000 at 4.5 TB/s: two blocks a multiprocessor leave 64 registers, of which 322 bytes are stored and 454 loaded,
//              and the loads are what it waits for
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/sslm_b200.h"
#include "sslm_cluster.cuh"
#include "sslm_kernels.h"

namespace sslm {
namespace {

constexpr int kMostWarps = 32;                // of a block of T threads (512: 1,024 a multiprocessor took 21 rows from 13.8 to 17.8 us)
constexpr int kList = 8192;                   // tokens of a row's list
constexpr int kSteps = 1024;                  // sums of 256 tokens
constexpr int kCounts = 2048;                 // places that a sample is counted into
constexpr int kPlaces = 512;                  // places that a selection counts into, four words each
constexpr int kIndexBits = kSampleIndexBits;  // of a token
constexpr int kMostVocab = kSampleMostVocab;
constexpr int kMostSlice = (kSteps - 2) * 256;      // a sum for every 256 tokens, and for the ends
constexpr int kMostBlocks = 16;
constexpr uint32_t kLate = 0xFFFFFFFFu;
// exchanges, in order: maxima and bounds; sums and lists' lengths; the lists; and where the list is too short the window's ends, its sums, its
// lists, the last key that is kept, sums and numbers of what is kept
// (a window's sums take two exchanges in turn, where one window is not enough)
enum { kTop = 0, kSums, kLists, kEnds, kWindow, kWindowLists, kBound, kKept, kWindowOdd, kBars };

struct SampleArgs {
	int rows, vocab, sub, slice;        // a row is cut over `sub` blocks of `slice` tokens (a multiple of 128)
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
// (of d up to `most`; beyond, anything)
__device__ __forceinline__ uint32_t weight_near(uint32_t d, const Scaled& s) {
	const uint32_t t = __umulhi(d << s.a, s.m) >> s.b, f = t << 8;
	uint32_t p = 14555373u;
	p = 114090822u - __umulhi(f, p);
	p = 514119776u - __umulhi(f, p);
	p = 1488326151u - __umulhi(f, p);
	p = 2147483648u - __umulhi(f, p);
	return __funnelshift_rc(p, 0u, t >> 24);
}
__device__ __forceinline__ uint32_t weight_of(uint32_t d, const Scaled& s) {
	const uint32_t p = weight_near(d, s);
	return d <= s.most ? p : 0u;
}
// the largest d with a weight of `least` or more (at most 2^31), by a warp: 32 places at a time
__device__ __forceinline__ uint32_t farthest_with(uint32_t least, const Scaled& s) {
	const uint32_t lane = threadIdx.x & 31;
	uint32_t low = 0, high = s.most;
	while (low < high) {
		const uint32_t span = high - low;
		const uint32_t d = span <= 32u ? low + 1u + min(lane, span - 1u) : low + (uint32_t)((unsigned long long)span * (lane + 1u) >> 5);
		const int n = __popc(__ballot_sync(0xffffffffu, weight_near(d, s) >= least));      // (the first n: weights fall)
		const uint32_t in = __shfl_sync(0xffffffffu, d, max(n - 1, 0)), out = __shfl_sync(0xffffffffu, d, min(n, 31));
		if (n > 0) low = in;
		if (n < 32) high = out - 1u;
		else high = low;
	}
	return low;
}
// floor(total part / 2^bits), part <= 2^bits
__device__ __forceinline__ unsigned long long share_of(unsigned long long total, uint32_t part, int bits) {
	const unsigned long long lo = total * part, hi = __umul64hi(total, part);
	return lo >> bits | hi << (64 - bits);
}

// ---- block-wide sums of numbers below 2^52 (2^20 weights of at most 2^31); s: 2 * kMostWarps words
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {      // (two words of 26 bits: five shuffles of 64 bits took three times as long)
	const uint32_t low = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0x3FFFFFFu), high = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 26));
	return ((unsigned long long)high << 26) + low;
}
// both, and a barrier
template <int T>
__device__ __forceinline__ ulonglong2 block_sums(unsigned long long a, unsigned long long b, unsigned long long* s) {
	a = warp_sum(a);
	b = warp_sum(b);
	__syncthreads();
	if ((threadIdx.x & 31) == 0) {
		s[threadIdx.x >> 5] = a;
		s[kMostWarps + (threadIdx.x >> 5)] = b;
	}
	__syncthreads();
	const int lane = threadIdx.x & 31;
	return ulonglong2{warp_sum(lane < T / 32 ? s[lane] : 0ull), warp_sum(lane < T / 32 ? s[kMostWarps + lane] : 0ull)};
}
// the sum of v over the threads in front of this one
__device__ __forceinline__ unsigned long long block_before(unsigned long long v, unsigned long long* s) {
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	unsigned long long upto = v;
#pragma unroll
	for (int o = 1; o < 32; o *= 2) {
		const unsigned long long z = __shfl_up_sync(0xffffffffu, upto, o);
		if (lane >= o) upto += z;
	}
	if (lane == 31) s[warp] = upto;
	__syncthreads();
	return upto - v + warp_sum(lane < warp ? s[lane] : 0ull);
}

// ---- elements of a row: those of a list, or all that have a weight. Their keys are d 2^20 + v.
struct Elements {
	const unsigned long long* list;
	unsigned long long origin;      // of the list's keys: they are (INT32_MAX - x) 2^20 + v
	const int32_t* logits;
	int n, vocab;
	int32_t top;
	Scaled scale;
	uint32_t floor_w;
};
template <int T, bool WHOLE, typename F>
__device__ __forceinline__ void each_key(const Elements& e, F f) {
	const int t = threadIdx.x;
	if (!WHOLE) {
		for (int i = t; i < e.n; i += T) f(e.list[i] - e.origin);
		return;
	}
	const int head = min(e.vocab, (int)((4 - (((uintptr_t)e.logits >> 2) & 3)) & 3)), words = (e.vocab - head) >> 2;
	auto one = [&](int32_t x, int v) {
		const uint32_t d = (uint32_t)e.top - (uint32_t)x;
		if (d <= e.scale.most) f((unsigned long long)d << kIndexBits | (uint32_t)v);
	};
	const int4* q = (const int4*)(e.logits + head);
#pragma unroll 1
	for (int k = t; k < words; k += 4 * T) {
		int4 y[4];
#pragma unroll
		for (int u = 0; u < 4; ++u)
			if (k + u * T < words) y[u] = __ldcg(q + k + u * T);
#pragma unroll
		for (int u = 0; u < 4; ++u) {
			if (k + u * T >= words) break;
			const int v = head + 4 * (k + u * T);
			one(y[u].x, v);
			one(y[u].y, v + 1);
			one(y[u].z, v + 2);
			one(y[u].w, v + 3);
		}
	}
	if (t < head) one(e.logits[t], t);
	const int behind = head + 4 * words + t;
	if (behind < e.vocab) one(e.logits[behind], behind);
}
__device__ __forceinline__ uint32_t key_weight(unsigned long long key, const Elements& e) { return weight_of((uint32_t)(key >> kIndexBits), e.scale); }

// ---- selection: the first element, by rising keys (by rising index: kByIndex), up to which, itself included, more than `target` of the
// weights lies (of the elements: kOnes), among those up to `bound` (and, by index, not below floor_w); their sum is above target. The elements are
// counted into 512 places by their keys' leading bits, those of the place that holds the one looked for again, until a place has at most 32.
// A place's sum is kept in three parts of 11 bits of each weight, for 2^20 elements in words of 32.
enum { kOnes = 0, kWeights, kByIndex };
constexpr int kFew = 64;
struct SelectSmem {
	unsigned long long key[32], scan[2 * kMostWarps], target, found;
	uint32_t weight[32], place, count, n;
	unsigned long long few_key[kFew];
	uint32_t few_weight[kFew], few_kept[kFew];
	int token;
	uint32_t token_weight;
};
template <int T, bool WHOLE>
__device__ __noinline__ unsigned long long select_key(const Elements& e, int what, unsigned long long bound, int bits, unsigned long long target, uint32_t* places, SelectSmem& s) {
	const int t = threadIdx.x, lane = t & 31;
	uint32_t* number = places + 3 * kPlaces;
	unsigned long long low = 0;
	auto each = [&](auto f) {
		each_key<T, WHOLE>(e, [&](unsigned long long key) {
			if (key > bound) return;
			const uint32_t w = what == kOnes ? 1u : key_weight(key, e);
			if (what == kByIndex) {
				if (w < e.floor_w) return;
				key &= kMostVocab - 1;
			}
			f(key, w);
		});
	};
	for (;;) {
		const int down = max(0, bits - 9);
		for (int i = t; i < 4 * kPlaces; i += T) places[i] = 0u;
		if (t == 0) s.n = 0u;
		__syncthreads();
		each([&](unsigned long long key, uint32_t w) {
			const unsigned long long i = (key - low) >> down;
			if (key < low || i >= (unsigned long long)kPlaces) return;
			uint32_t* p = places + (int)i;
			atomicAdd(p + 3 * kPlaces, 1u);
			if (what == kOnes) return;
			atomicAdd(p, w & 0x7FFu);
			atomicAdd(p + kPlaces, w >> 11 & 0x7FFu);
			atomicAdd(p + 2 * kPlaces, w >> 22);
		});
		__syncthreads();
		const unsigned long long v = t >= kPlaces ? 0ull : what == kOnes ? (unsigned long long)number[t] : ((unsigned long long)places[2 * kPlaces + t] << 22) + ((unsigned long long)places[kPlaces + t] << 11) + places[t];
		const unsigned long long before = block_before(v, s.scan);
		if (before <= target && target < before + v) {      // (one thread's place)
			s.place = t;
			s.count = number[t];
			s.target = target - before;
		}
		__syncthreads();
		low += (unsigned long long)s.place << down;
		target = s.target;
		const uint32_t n = s.count;
		if (n <= 32u) {
			each([&](unsigned long long key, uint32_t w) {
				if (key < low || (key - low) >> down != 0ull) return;
				const uint32_t i = atomicAdd(&s.n, 1u);
				s.key[i] = key;
				s.weight[i] = w;
			});
			__syncthreads();
			if (t < 32) {
				const unsigned long long key = lane < n ? s.key[lane] : ~0ull;
				const uint32_t w = lane < n ? s.weight[lane] : 0u;
				unsigned long long less = 0;
				for (uint32_t i = 0; i < n; ++i)
					if (s.key[i] < key) less += s.weight[i];
				if (less <= target && target < less + w) s.found = key;
			}
			__syncthreads();
			return s.found;
		}
		bits = down;      // (keys differ, so a place of one key has one element)
	}
}

struct Drawn {
	int token;
	uint32_t weight, number;
	unsigned long long sum;
};
// The draw from at most 64 elements (s.few_key, `few` of them), cut by top-p (of `sum`, or of their own sum where that is 0) and min-p: eight threads an
// element compare it with eight others each. For 512 threads at least.
__device__ __noinline__ Drawn draw_few(const Elements& e, int few, uint32_t top_p, uint32_t draw, unsigned long long sum, SelectSmem& s) {
	const int t = threadIdx.x, i = t >> 3;
	if (t < kFew) {
		if (t >= few) s.few_key[t] = ~0ull;
		s.few_weight[t] = t < few ? key_weight(s.few_key[t], e) : 0u;
	}
	__syncthreads();
	auto eighth = [](unsigned long long v) {
#pragma unroll
		for (int o = 1; o < 8; o *= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
		return v;
	};
	const unsigned long long key = i < kFew ? s.few_key[i] : ~0ull;
	const uint32_t w = i < kFew ? s.few_weight[i] : 0u;
	unsigned long long less = 0, all = 0;
#pragma unroll
	for (int j = t & 7; j < kFew; j += 8) {
		all += s.few_weight[j];
		less += s.few_key[j] < key ? s.few_weight[j] : 0u;
	}
	less = eighth(less);
	all = eighth(all);
	const unsigned long long enough = top_p < (1u << 30) ? share_of(sum != 0ull ? sum : all, top_p, 30) : ~0ull;
	const bool kept = less < enough && w >= e.floor_w;
	if (i < kFew && (t & 7) == 0) s.few_kept[i] = kept ? w : 0u;
	__syncthreads();
	uint32_t number = 0;
	const uint32_t v = (uint32_t)key & (kMostVocab - 1);
	less = all = 0;
#pragma unroll
	for (int j = t & 7; j < kFew; j += 8) {
		const uint32_t g = s.few_kept[j];
		all += g;
		number += min(g, 1u);
		less += ((uint32_t)s.few_key[j] & (kMostVocab - 1)) < v ? g : 0u;
	}
	less = eighth(less);
	all = eighth(all);
#pragma unroll
	for (int o = 1; o < 8; o *= 2) number += __shfl_xor_sync(0xffffffffu, number, o);
	const unsigned long long mark = share_of(all, draw, 31);
	if (kept && (t & 7) == 0 && less <= mark && mark < less + w) {      // (one thread)
		s.token = (int)v;
		s.token_weight = w;
	}
	__syncthreads();
	return Drawn{s.token, s.token_weight, number, all};
}
// What a row's elements are cut to, and the token drawn from them. sum: of all weights, where top-k does not say what counts.
template <int T, bool WHOLE>
__device__ __forceinline__ Drawn draw_from(const Elements& e, int top_k, uint32_t top_p, uint32_t draw, unsigned long long sum, uint32_t* places, SelectSmem& s) {
	const int t = threadIdx.x, bits = kIndexBits + 32 - __clz((int)e.scale.most);
	unsigned long long bound = ~0ull;      // the last key that is kept
	auto take_few = [&]() {                // the elements up to it
		if (t == 0) s.n = 0u;
		__syncthreads();
		each_key<T, WHOLE>(e, [&](unsigned long long key) {
			if (key <= bound) s.few_key[atomicAdd(&s.n, 1u)] = key;
		});
		__syncthreads();
	};
	if (top_k > 0) {
		unsigned long long have = (unsigned long long)e.n, x = 0;
		if (WHOLE) {
			each_key<T, WHOLE>(e, [&](unsigned long long) { ++x; });
			have = block_sums<T>(x, 0ull, s.scan).x;
		}
		if (have > (unsigned long long)top_k) bound = select_key<T, WHOLE>(e, kOnes, bound, bits, (unsigned long long)top_k - 1ull, places, s);
		have = min(have, (unsigned long long)top_k);
		if (have <= (unsigned long long)kFew) {
			take_few();
			return draw_few(e, (int)have, top_p, draw, 0ull, s);
		}
		if (top_p < (1u << 30)) {
			x = 0;
			each_key<T, WHOLE>(e, [&](unsigned long long key) { x += key <= bound ? key_weight(key, e) : 0u; });
			sum = block_sums<T>(x, 0ull, s.scan).x;
		}
	}
	// (the sum is 2^31 at least, so the share is 2 at least)
	if (top_p < (1u << 30)) bound = select_key<T, WHOLE>(e, kWeights, bound, bits, share_of(sum, top_p, 30) - 1ull, places, s);
	unsigned long long mass = 0, many = 0;
	each_key<T, WHOLE>(e, [&](unsigned long long key) {
		if (key > bound) return;
		const uint32_t g = key_weight(key, e);
		many += 1ull << 32;
		if (g < e.floor_w) return;
		mass += g;
		++many;
	});
	const ulonglong2 all = block_sums<T>(mass, many, s.scan);
	if (all.y >> 32 <= (unsigned long long)kFew) {
		take_few();
		return draw_few(e, (int)(all.y >> 32), top_p, draw, sum, s);
	}
	const int token = (int)select_key<T, WHOLE>(e, kByIndex, bound, kIndexBits, share_of(all.x, draw, 31), places, s);
	return Drawn{token, weight_of((uint32_t)e.top - (uint32_t)e.logits[token], e.scale), (uint32_t)all.y, all.x};
}

struct SampleSmem {
	// keys of the list [kList], sums of 256 tokens [kSteps], counts [kCounts], the block's logits [slice] if they are kept
	static size_t bytes(int keep, int slice) { return (size_t)kList * 8 + (size_t)kSteps * 8 + (size_t)kCounts * 4 + (keep ? (size_t)slice * 4 + 16 : 0); }
};

template <bool RESIDENT, bool KEEP, int T, int BLOCKS>
__global__ void __launch_bounds__(T, BLOCKS) k_sample(const __grid_constant__ SampleArgs a) {
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ __align__(8) unsigned long long s_bar[kBars], s_sum[3][kMostBlocks], s_listed[3][kMostBlocks], s_bound;
	__shared__ int2 s_top[kMostBlocks], s_warp[kMostWarps], s_ends;
	__shared__ uint32_t s_count[3][kMostBlocks], s_n, s_kept_far;
	__shared__ Row s_row;
	__shared__ SelectSmem s_select;
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.vocab;
	const int sub = a.sub, rank = (int)blockIdx.x;
	const int64_t r = blockIdx.y;
	unsigned long long *list = (unsigned long long*)smem, *steps = list + kList, *scan = s_select.scan;
	uint32_t* counts = (uint32_t*)(steps + kSteps);
	int4* kept = (int4*)(counts + kCounts);
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
	const int32_t* const logits = RESIDENT ? a.logits + r * a.logits_stride : a.desc[r].logits;
	if (!RESIDENT && logits == nullptr) {      // (a row that is not sampled; all blocks of the cluster alike)
		if (sub > 1) cluster_wait();
		return;
	}
	int32_t p[6] = {0, 0, 0, 1, 0, 0};         // asked for here, looked at behind the first pass
	SampleRow d{};
	Scale in{0, 0};
	if (t == 0) {
		if (RESIDENT) {
#pragma unroll
			for (int i = 0; i < 5; ++i) p[i] = a.params[5 * r + i];
			p[5] = a.draws[r];
		} else {
			d = a.desc[r];
			in = a.scales[r];
		}
	}
	auto take_record = [&]() {
		if (t != 0) return;
		Row x{};
		x.logits = logits;
		if (RESIDENT) {
			if (p[0] < 0 || p[1] < 0 || p[1] > 63 || p[2] < 0 || p[3] < 1 || p[3] > (1 << 30) || p[4] < 0 || p[4] > (1 << 30) || p[5] < 0) x.code = SSLM_B200_ROW_CONSTANTS;
			x.slope = (uint32_t)p[0]; x.cut = (uint32_t)p[1]; x.draw = (uint32_t)p[5];
			x.top_k = p[2]; x.top_p = (uint32_t)p[3]; x.min_p = (uint32_t)p[4];
			if (rank == 0 && a.status != nullptr) a.status[r] = x.code;
		} else {
			// octaves a logit unit: the sequence's constant times the scale of the row that the head multiplied
			const Scale s = combine(Scale{d.slope_m, d.slope_e}, in);
			const int64_t cut = -(s.e + 24);
			x.slope = cut < 0 ? 1u << 30 : (cut > 94 ? 0u : (uint32_t)s.m >> (cut > 63 ? (int)cut - 63 : 0));      // (64 octaves a unit are as good as more)
			x.cut = (uint32_t)max((int64_t)0, min((int64_t)63, cut));
			x.draw = d.draw;
			x.top_k = d.top_k; x.top_p = d.top_p; x.min_p = d.min_p;
			x.layer = d.layer;
		}
		s_row = x;
	};
	const int s0 = min(V, rank * a.slice), s1 = min(V, s0 + a.slice);
	// four neighbouring tokens lie in one aligned 16-byte word: whole words from `first` to `last`, the ends token by token
	const int mis = (int)(((uintptr_t)logits >> 2) & 3);
	const int first = min(s1, s0 + ((4 - ((s0 + mis) & 3)) & 3)), words = (s1 - first) >> 2, last = first + 4 * words;
	const int4* from = (const int4*)(logits + first);
	const int heads = first - s0, tails = s1 - last;
	const int end = t < heads ? s0 + t : (t >= 4 && t - 4 < tails ? last + t - 4 : -1);      // the token of the ends that is this thread's
	const int32_t end_x = end >= 0 ? logits[end] : INT32_MIN;
	auto top_of = [&](int4 q) { return max(max(q.x, q.y), max(q.z, q.w)); };
	auto at_least = [&](int4 q, int32_t least) { return (q.x >= least ? 1u : 0u) | (q.y >= least ? 2u : 0u) | (q.z >= least ? 4u : 0u) | (q.w >= least ? 8u : 0u); };
	// Room in the list for the tokens that a lane's `which` names: one atomic a lane that has any, asked for a round before its place is needed. (One
	// a warp, with the lanes' places from ballots: 64 rows with top-p 97 us instead of 91, with top-k 27 instead of 24. One a token, waited for: more.)
	auto reserve = [&](uint32_t which) { return which != 0u ? atomicAdd(&s_n, (uint32_t)__popc(which)) : 0u; };
	auto put = [&](uint32_t at, int32_t x, int v) {
		if (at < (uint32_t)kList) list[at] = (unsigned long long)(0x7FFFFFFFu - (uint32_t)x) << kIndexBits | (uint32_t)v;
	};
	auto pick = [](const auto (&v)[8], int j) {      // v[j] of registers
		const auto a = (j & 1) != 0 ? v[1] : v[0], b = (j & 1) != 0 ? v[3] : v[2], c = (j & 1) != 0 ? v[5] : v[4], d = (j & 1) != 0 ? v[7] : v[6];
		return (j & 4) != 0 ? ((j & 2) != 0 ? d : c) : ((j & 2) != 0 ? b : a);
	};
	auto put_end = [&]() {
		put(atomicAdd(&s_n, 1u), end_x, end);
	};
	// a wait ran out: the row is reported, and the block stays until nothing can be sent to it any more
	auto give_up = [&](bool stay) {
		if (t == 0) {
			if (RESIDENT) {
				if (a.status != nullptr) a.status[r] = kInternalWaitTimeout;
			} else {
				atomicCAS(&a.status[r], 0, pack_status(kInternalWaitTimeout, kSiteLogits, s_row.layer));
			}
		}
		if (stay) exchange_leave(cta_addr(&s_bar[0]), kBars);
	};

	// ---- the maximum, and the least of the groups' maxima
	int32_t top = end_x;
	bool early = false;
	int32_t early_least = INT32_MIN;
	if (!KEEP && sub == 1) {
		take_record();
		__syncthreads();
		// One block has a long row and a small top-k: the least of the maxima of the row's first eighth, of 16 to 64 groups, leaves eight times as
		// many tokens of the row as of that eighth, so the list can be made in the first pass already (256 rows: a pass less).
		const int top_k = s_row.top_k;
		early = s_row.code == 0 && top_k > 0 && top_k <= 400 && words >= 16 * T;
		if (early) {
			int32_t m = INT32_MIN;
			const int part = words / (8 * T) * T;
#pragma unroll 4
			for (int k = t; k < part; k += T) m = max(m, top_of(__ldcg(from + k)));
			const int mates = top_k <= 64 ? 32 : (top_k <= 160 ? 16 : 8);      // threads of a group
			for (int o = 1; o < mates; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
			m = __reduce_min_sync(0xffffffffu, m);
			if (lane == 0) s_warp[warp] = make_int2(m, 0);
			__syncthreads();
			early_least = max(INT32_MIN + 1, __reduce_min_sync(0xffffffffu, s_warp[lane & (T / 32 - 1)].x));
			if (end_x >= early_least) put_end();
		}
	}
	{
		constexpr int U = 4;
		int4 q[U], y[U];
		auto fetch = [&](int4 (&to)[U], int k) {
#pragma unroll
			for (int u = 0; u < U; ++u) {
				to[u] = make_int4(INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN);
				if (k + u * T < words) to[u] = __ldcg(from + k + u * T);
			}
		};
		fetch(q, t);
#pragma unroll 1
		for (int k = t; k - t < words; k += U * T) {
			fetch(y, k + U * T);
			uint32_t which = 0;
#pragma unroll
			for (int u = 0; u < U; ++u) {
				if (KEEP && k + u * T < words) kept[k + u * T] = q[u];
				const int32_t m = top_of(q[u]);
				top = max(top, m);
				if (!KEEP && early && m >= early_least) which |= at_least(q[u], early_least) << (4 * u);
				q[u] = y[u];
			}
			if (!KEEP && early) {      // (few: read again)
				uint32_t at = reserve(which);
#pragma unroll 1
				for (; which != 0u; which &= which - 1u, ++at) {
					const int j = __ffs((int)which) - 1, i = 4 * (k + (j >> 2) * T) + (j & 3);
					put(at, __ldcg(logits + first + i), first + i);
				}
			}
		}
	}
	if (KEEP || sub > 1) take_record();      // (it arrived meanwhile)
	__syncthreads();
	const Row w = s_row;
	if (w.code != 0) {      // (all blocks of the cluster alike)
		if (sub > 1) cluster_wait();
		return;
	}
	const bool cuts = w.top_k > 0 || w.top_p < (1u << 30);
	int32_t least = INT32_MAX;
	int group = 1;      // threads of a group, over all blocks 256 groups or more, or as many as there are tokens to keep
	if (cuts) {
		int wanted = 256;
		if (w.top_k > 0) {
			wanted = 32;
			while (wanted < min(w.top_k, 512)) wanted *= 2;
		}
		while (group < T && 2 * group * wanted <= sub * T) group *= 2;
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
		const int2 x = s_warp[lane & (T / 32 - 1)];
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
	const uint32_t floor_w = max(1u, 2u * w.min_p);
	if (warp == T / 32 - 1 && w.top_k == 0) {      // (beside the exchange; the largest logit only makes it less)
		const uint32_t d = farthest_with(floor_w, scaled_of(w.slope, w.cut, INT32_MAX));
		if (lane == 0) s_kept_far = d;
	}
	if (sub == 1) __syncthreads();
	if (sub > 1) {
		cluster_wait();      // (all blocks run)
		if (t < sub) exchange_send(&s_top[rank], cta_addr(&s_bar[kTop]), (uint32_t)t, make_int2(top, least));
		late = !exchange_wait(cta_addr(&s_bar[kTop]));
		const int2 x = lane < sub ? s_top[lane] : make_int2(INT32_MIN, INT32_MAX);
		top = __reduce_max_sync(0xffffffffu, x.x);
		least = __reduce_min_sync(0xffffffffu, x.y);
		late = __syncthreads_or(late) != 0;
	}
	const bool none = top == INT32_MIN;
	const Scaled scale = scaled_of(w.slope, w.cut, none ? INT32_MAX : top);
	const uint32_t most = scale.most;
	auto weight = [&](int32_t x) { return weight_of((uint32_t)top - (uint32_t)x, scale); };      // (0 of INT32_MIN)
	auto x_of = [&](uint32_t d) { return (int32_t)max((long long)top - (long long)d, -2147483647ll); };      // the logit that lies d below the largest
	const uint32_t reach = least == INT32_MIN ? 0xFFFFFFFFu : (uint32_t)top - (uint32_t)max(least, INT32_MIN + 1), far = min(reach, most);      // the list's farthest
	bool complete = reach >= most;      // the list has every token that has a weight
	bool have_list = false;
	if (early) {      // (of no use where some of its tokens have no weight: they do not count)
		have_list = s_n >= (uint32_t)w.top_k && s_n <= (uint32_t)kList && (uint32_t)top - (uint32_t)early_least <= most;
		__syncthreads();      // (all have seen how long it is)
		if (have_list) complete = false;
		else if (t == 0) s_n = 0u;
	}

	// ---- passes: the second one, and those over a window. A pass adds up the weights of the logits from near_x on (sum), and, where there are sums of
	// 256 neighbouring tokens (the ends at steps[0] and steps[last_step]), what is kept of them; it lists the logits from from_x on, with those sums only
	// the ones below near_x, and adds up their weights (listed).
	const int last_step = (words + 63) / 64 + 1;
	unsigned long long sum = 0, listed = 0, kept_sum = 0;
	uint32_t count = 0, kept_count = 0, others = 0, total = 0;      // tokens of the block's list, of what it keeps, of lower blocks' lists, of all lists
	// sums of all blocks; false where a wait ran out here or elsewhere
	auto tell = [&](int bar, int slot, bool both, uint32_t turn) {
		if (t < sub) {
			exchange_send(&s_sum[slot][rank], cta_addr(&s_bar[bar]), (uint32_t)t, sum);
			if (both) exchange_send(&s_listed[slot][rank], cta_addr(&s_bar[bar]), (uint32_t)t, listed);
			exchange_send(&s_count[slot][rank], cta_addr(&s_bar[bar]), (uint32_t)t, late ? kLate : count);
		}
		const bool waited = bounded_wait<true>(cta_addr(&s_bar[bar]), turn & 1u);
		const bool gave_up = __syncthreads_or(late || !waited) != 0;
		if (__any_sync(0xffffffffu, lane < sub && s_count[slot][min(lane, sub - 1)] == kLate) || gave_up) {
			give_up(gave_up || rank == 0);
			return false;
		}
		return true;
	};
	auto add_up = [&](int slot, bool both) {
		sum = listed = 0;
		others = total = 0;
		for (int i = 0; i < sub; ++i) {
			sum += s_sum[slot][i];
			if (both) listed += s_listed[slot][i];
			if (i < rank) others += s_count[slot][i];
			total += s_count[slot][i];
		}
	};
	// with windows: what is kept ends at a d in (begin, stop], up to which exactly `before_begin` and `through_stop` of the weights lie; near < d <= until
	// is the window, `sure` lies in front of it
	uint32_t begin = far, stop = most, near = 0, until = far, turn = 0;
	unsigned long long before_begin = 0, through_stop = 0, all_weights = 0, enough = 0, sure = 0;
	const bool weigh = w.top_k == 0;      // (of a row with top-k the list alone)
	bool by_steps = !cuts, wide = false, fits = false;
#pragma unroll 1
	for (;;) {
		const int32_t near_x = turn == 0u ? INT32_MIN + 1 : x_of(near), from_x = x_of(until);
		const int32_t first_x = turn == 0u ? x_of(most) : near_x, kept_x = max(first_x, x_of(s_kept_far));      // what is added up, and what of it is kept
		unsigned long long first_sum = 0, in_list = 0;
		uint32_t many = 0;
		if (by_steps && t < 2) steps[t == 0 ? 0 : last_step] = 0ull;
		__syncthreads();
		if (!late && !none && !have_list) {
			if (weigh && end_x >= near_x) {
				const uint32_t g = weight(end_x);
				first_sum += g;
				if (by_steps && end_x >= kept_x) {
					++many;
					atomicAdd(&steps[t < 4 ? 0 : last_step], (unsigned long long)g);
				}
			}
			if (cuts && end_x >= from_x && !(by_steps && end_x >= near_x)) {
				in_list += weight(end_x);
				put_end();
			}
			// (two neighbouring words a thread and round, from the last ones on: what was read last is likelier still in L2)
			const int rounds = (words + 2 * T - 1) / (2 * T);
			auto fetch = [&](int k) { return (uint32_t)k < (uint32_t)words ? (KEEP ? kept[k] : __ldcg(from + k)) : make_int4(INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN); };
			auto wanted = [&](int4 u, int4 v) {      // of the list
				if (!cuts || max(top_of(u), top_of(v)) < from_x) return 0u;
				const uint32_t in = at_least(u, from_x) | at_least(v, from_x) << 4;
				return by_steps ? in & ~(at_least(u, near_x) | at_least(v, near_x) << 4) : in;
			};
			int k = 2 * ((rounds - 1) * T + t);
			int4 q0 = fetch(k), q1 = fetch(k + 1);
			uint32_t which = wanted(q0, q1), at = reserve(which);
#pragma unroll 1
			for (int i = 0; i < rounds; ++i, k -= 2 * T) {
				int4 y0 = q0, y1 = q1;
				if (i + 1 < rounds) {
					y0 = KEEP ? kept[k - 2 * T] : __ldcg(from + k - 2 * T);
					y1 = KEEP ? kept[k - 2 * T + 1] : __ldcg(from + k - 2 * T + 1);
				}
				const int32_t x[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
				uint32_t g[8];
				if (weigh) {
#pragma unroll
					for (int j = 0; j < 8; ++j) g[j] = weight_near((uint32_t)top - (uint32_t)x[j], scale);
					if (cuts) {
#pragma unroll
						for (int j = 0; j < 8; ++j) first_sum += x[j] >= first_x ? g[j] : 0u;
					}
					if (by_steps) {
						unsigned long long s8 = 0;
#pragma unroll
						for (int j = 0; j < 8; ++j) {
							const bool yes = x[j] >= kept_x;
							s8 += yes ? g[j] : 0u;
							if (yes) ++many;
						}
						const uint32_t high = __reduce_add_sync(0xffffffffu, (uint32_t)(s8 >> 16)), low = __reduce_add_sync(0xffffffffu, (uint32_t)s8 & 0xFFFFu);
						if (lane == 0 && k < words) steps[1 + (k >> 6)] = ((unsigned long long)high << 16) + low;
					}
				}
				if (cuts) {      // (few, a lane seldom has two: one at a time, by choosing, took 64 rows with top-p from 91 to 80 us)
#pragma unroll 1
					for (; which != 0u; which &= which - 1u, ++at) {
						const int j = __ffs((int)which) - 1;
						put(at, pick(x, j), first + 4 * k + j);
						if (weigh) in_list += pick(g, j);
					}
					which = i + 1 < rounds ? wanted(y0, y1) : 0u;
					at = reserve(which);
				}
				q0 = y0;
				q1 = y1;
			}
			__syncthreads();
		}
		// ---- sums over the block (behind which its list is whole), and over all blocks
		if (by_steps) {
			kept_sum = 0;
			if (!none && !late)
				for (int i = t; i <= last_step; i += T) kept_sum += steps[i];
			const ulonglong2 both = block_sums<T>(kept_sum, many, scan);
			kept_sum = both.x;
			kept_count = (uint32_t)both.y;
		}
		{
			const ulonglong2 both = block_sums<T>(first_sum, in_list, scan);
			sum = cuts ? both.x : kept_sum;
			listed = both.y;
			count = total = cuts ? s_n : kept_count;
		}
		if (sub > 1) {
			const int slot = turn == 0u ? 0 : 2 - (int)(turn & 1u), bar = slot == 0 ? kSums : (slot == 1 ? kWindow : kWindowOdd);
			if (!tell(bar, slot, true, turn == 0u ? 0u : (turn - 1u) >> 1)) return;
			add_up(slot, true);
		}
		if (!cuts || none) break;
		if (turn == 0u) {
			all_weights = sum;
			enough = weigh ? share_of(sum, w.top_p, 30) : 0ull;
			fits = total <= (uint32_t)kList && (complete || (weigh ? listed >= enough : total >= (uint32_t)w.top_k));
			wide = !fits && weigh && total <= (uint32_t)kList;
			if (!wide) break;
			by_steps = true;
			before_begin = listed;
			through_stop = sum;
		} else {
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
			wide = turn < 6u && stop - begin > 1u;
			if (!wide) break;
			if (sub > 1 && t == 0) {      // (of the next turn's ends and the next but one's sums; what comes may have come already)
				asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(cta_addr(&s_bar[(turn & 1u) != 0u ? kWindow : kWindowOdd])), "r"((uint32_t)(sub * 20)) : "memory");
				if (rank != 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(cta_addr(&s_bar[kEnds])), "r"(8u) : "memory");
			}
			__syncthreads();
		}
		// ---- a window. A sample (32,768 to 65,536 of the first block's tokens, or all) says where between begin and stop, to one or two in a hundred; the
		// window is three to either side, or less where that would be too many tokens
		if (rank == 0) {
			const int down = max(0, 32 - __clz((int)(stop - begin)) - 11);
			for (int i = t; i < kCounts; i += T) counts[i] = 0u;
			__syncthreads();
			const int every = max(1, words / 8192);
#pragma unroll 2
			for (int k = t * every; k < words; k += T * every) {
				const int4 q = KEEP ? kept[k] : __ldcg(from + k);
				const int32_t y[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
				for (int j = 0; j < 4; ++j) {
					const uint32_t d = (uint32_t)top - (uint32_t)y[j];
					if (d > begin && d <= stop) atomicAdd(&counts[min((d - begin - 1u) >> down, (uint32_t)kCounts - 1u)], 1u);
				}
			}
			__syncthreads();
			// weights of the places, in units such that none is above 2^15 (and no place's sum above 2^31)
			const int shift = max(0, 17 - __clz((int)weight_of(begin, scale)));
			constexpr int N = kCounts / T;
			unsigned long long v[N], at = 0;
#pragma unroll
			for (int j = 0; j < N; ++j) {
				const uint32_t i = N * t + j, mid = begin + 1u + (i << down) + ((1u << down) >> 1);
				v[j] = mid > begin ? (unsigned long long)(counts[i] * (weight_of(mid, scale) >> shift)) : 0ull;
				at += v[j];
			}
			const unsigned long long all = block_sums<T>(at, 0ull, scan).x;
			__syncthreads();
			at = block_before(at, scan);
			const double want = (double)(enough - before_begin) / (double)(through_stop - before_begin);
			double slack = 0.03;
#pragma unroll 1
			for (int trial = 0; trial < 2; ++trial) {
				const double low = (want - slack) * (double)all, high = (want + slack) * (double)all;
				if (t == 0) s_ends = make_int2((int)begin, (int)stop);
				__syncthreads();
				unsigned long long in = 0, z = at;
#pragma unroll
				for (int j = 0; j < N; ++j) {
					const uint32_t i = N * t + j;
					if ((double)z <= low && low < (double)(z + v[j])) s_ends.x = (int)(begin + (i << down));
					if ((double)z <= high && high < (double)(z + v[j])) s_ends.y = (int)min((unsigned long long)stop, (unsigned long long)begin + ((unsigned long long)(i + 1) << down));
					if ((double)(z + v[j]) > low && (double)z <= high) in += counts[i];
					z += v[j];
				}
				in = block_sums<T>(in, 0ull, scan).x * (unsigned long long)(every * sub);      // tokens of the row that are to be expected
				if (in <= (unsigned long long)kList * 3 / 4) break;
				slack = max(0.01, slack * (double)(kList / 2) / (double)in);
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
		near = (uint32_t)s_ends.x;
		until = (uint32_t)s_ends.y;
		if (t == 0) s_n = 0u;
		++turn;
	}
	Drawn out{-2, 0u, 0u, 0ull};
	unsigned long long bound = ~0ull;      // the last key that is kept
	if (cuts) by_steps = false;
	if (cuts && !none) {
		const unsigned long long origin = (unsigned long long)(0x7FFFFFFFu - (uint32_t)top) << kIndexBits;
		if (!fits && !wide && rank != 0) return;
		const uint32_t own_listed = count;      // (at the front of the list)
		if (sub > 1 && (fits || wide)) {        // the lists, to the first block
			const uint32_t bar = cta_addr(&s_bar[wide ? kWindowLists : kLists]);
			if (rank != 0) {
				for (uint32_t i = t; i < count; i += T) exchange_send(list + others + i, bar, 0u, list[i]);
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
		const Elements e{list, origin, w.logits, (int)total, V, top, scale, floor_w};
		if (wide) {
			if (rank == 0) {
				bound = select_key<T, false>(e, kWeights, ~0ull, kIndexBits + 32 - __clz((int)most), enough - 1ull - sure, counts, s_select);
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
			// the block's tokens of the window that are kept, to the sums of their 256 neighbours
			sum = 0;
			count = 0;
			for (uint32_t i = t; i < own_listed; i += T) {
				const unsigned long long key = list[i] - origin;
				const uint32_t g = key_weight(key, e);
				if (key > bound || g < floor_w) continue;
				const int v = (int)(key & (kMostVocab - 1));
				sum += g;
				++count;
				atomicAdd(&steps[v < first ? 0 : (v >= last ? last_step : 1 + ((v - first) >> 8))], (unsigned long long)g);
			}
			const ulonglong2 both = block_sums<T>(sum, count, scan);
			sum = both.x + kept_sum;
			count = total = (uint32_t)both.y + kept_count;
			if (sub > 1) {
				if (!tell(kKept, 0, false, 0u)) return;
				add_up(0, false);
			}
			by_steps = true;
		} else if (fits) {
			out = draw_from<T, false>(e, w.top_k, w.top_p, w.draw, all_weights, counts, s_select);
		} else {
			out = draw_from<T, true>(e, w.top_k, w.top_p, w.draw, all_weights, counts, s_select);
		}
	}
	if (by_steps && !none) {
		// the block whose sums the mark lies in, the 256 tokens, then the token
		unsigned long long mark = share_of(sum, w.draw, 31);
		int owner = 0;
		if (sub > 1) {
			unsigned long long before = 0;
			for (int i = 0; i < sub; ++i) {
				if (before <= mark && mark < before + s_sum[0][i]) {
					owner = i;
					break;
				}
				before += s_sum[0][i];
			}
			mark -= before;
		}
		if (rank != owner) return;
		out.sum = sum;
		out.number = total;
		constexpr int N = kSteps / T;
		unsigned long long v[N], at = 0;
#pragma unroll
		for (int j = 0; j < N; ++j) {
			v[j] = N * t + j <= last_step ? steps[N * t + j] : 0ull;
			at += v[j];
		}
		__syncthreads();
		at = block_before(at, scan);
#pragma unroll
		for (int j = 0; j < N; ++j) {
			if (at <= mark && mark < at + v[j]) {
				s_select.place = N * t + j;
				s_select.target = mark - at;
			}
			at += v[j];
		}
		__syncthreads();
		if (warp != 0) return;
		const int step = (int)s_select.place;
		mark = s_select.target;
		const int v0 = step == 0 ? s0 : (step == last_step ? last : first + 256 * (step - 1)), v1 = step == 0 ? first : (step == last_step ? s1 : min(last, v0 + 256));
		uint32_t g[8];
		unsigned long long own = 0;
#pragma unroll
		for (int j = 0; j < 8; ++j) {
			const int i = v0 + 8 * lane + j;
			const int32_t x = i < v1 ? logits[i] : INT32_MIN;
			g[j] = weight(x);
			if (g[j] < floor_w || ((unsigned long long)((uint32_t)top - (uint32_t)x) << kIndexBits | (uint32_t)i) > bound) g[j] = 0u;
			own += g[j];
		}
		unsigned long long upto = own;
#pragma unroll
		for (int o = 1; o < 32; o *= 2) {
			const unsigned long long z = __shfl_up_sync(0xffffffffu, upto, o);
			if (lane >= o) upto += z;
		}
		unsigned long long before = upto - own;
		const int who = __ffs(__ballot_sync(0xffffffffu, before <= mark && mark < upto)) - 1;
#pragma unroll
		for (int j = 0; j < 8; ++j) {
			if (out.token < 0 && before <= mark && mark < before + g[j]) {
				out.token = v0 + 8 * lane + j;
				out.weight = g[j];
			}
			before += g[j];
		}
		out.token = __shfl_sync(0xffffffffu, out.token, who);
		out.weight = __shfl_sync(0xffffffffu, out.weight, who);
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

// Blocks a row: with few rows as many as leave every block a multiprocessor of its own (clusters do not fill the device: 132 of its 148), with
// slices of 4,096 tokens and more, else one. 64 rows of 151,936: two blocks 97 us with top-p and 27 with top-k (one 156 and 28, three 131 and 35, four
// 109 and 30, eight 133 and 48, as the kernel stood then); 32 rows: four 63 and 17 (two 92 and 23, eight 72 and 28).
void sample_plan(SampleArgs* a) {
	const int sms = sm_count(), most = std::max(1, (sms - 16) / a->rows), need = (a->vocab + kMostSlice - 128 - 1) / (kMostSlice - 128);
	a->sub = std::min(kMostBlocks, std::max(need, std::min(most, std::max(1, a->vocab / 4096))));
	a->slice = ((a->vocab + a->sub - 1) / a->sub + 127) & ~127;
	a->keep = a->rows * a->sub <= sms && SampleSmem::bytes(1, a->slice) <= (size_t)220 * 1024 ? 1 : 0;
}

template <bool RESIDENT, bool KEEP, int T, int BLOCKS>
cudaError_t sample_launch_as(SampleArgs a, cudaStream_t st) {
	static PerDeviceOnce once;
	const auto kernel = k_sample<RESIDENT, KEEP, T, BLOCKS>;
	cudaError_t e = once_per_device(once, [&] {
		const cudaError_t x = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
		return x != cudaSuccess ? x : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, KEEP ? 220 * 1024 : (int)SampleSmem::bytes(0, 0));
	});
	if (e != cudaSuccess) return e;
	a.debug_withhold = exchange_debug_take(kExchangeSample);
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3(a.sub, a.rows);
	cfg.blockDim = dim3(T);
	cfg.dynamicSmemBytes = SampleSmem::bytes(KEEP, a.slice);
	cfg.stream = st;
	cudaLaunchAttribute attr[2];
	attr[0].id = cudaLaunchAttributeClusterDimension;
	attr[0].val.clusterDim.x = (unsigned)a.sub;
	attr[0].val.clusterDim.y = 1;
	attr[0].val.clusterDim.z = 1;
	attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[1].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = attr;
	cfg.numAttrs = pdl_enabled() ? 2 : 1;
	return cudaLaunchKernelEx(&cfg, kernel, a);
}
template <bool RESIDENT>
cudaError_t sample_launch(const SampleArgs& a, cudaStream_t st) {
	if (a.keep) return sample_launch_as<RESIDENT, true, 512, 1>(a, st);
	return a.rows * a.sub <= sm_count() ? sample_launch_as<RESIDENT, false, 512, 1>(a, st) : sample_launch_as<RESIDENT, false, 512, 2>(a, st);
}

}  // namespace

cudaError_t launch_sample(const SampleRow* rows, int m, int vocab, const Scale* scales, unsigned long long* best, int32_t* status, cudaStream_t st) {
	SampleArgs a{};
	a.rows = m; a.vocab = vocab;
	a.desc = rows; a.scales = scales; a.best = best; a.status = status;
	sample_plan(&a);
	return sample_launch<false>(a, st);
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
	if (sample_launch<true>(a, (cudaStream_t)stream) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}
