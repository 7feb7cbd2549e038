// The pages of a cache on a caller's tensors: sequences that continue from others, grow or end (fork), and the pages in use moved to the
// front of the pool (compact). Both decide who holds which page, in one kernel of one cluster, and leave a list of pages to be copied, which a
// second kernel works off in every plane of the pool.
//
// Page ids are given out lowest first and in the order of the sequences, whatever order threads run in: ranks come from sums over ranges
// of pages and of sequences, a range to a block of the cluster; holders are counted with integer atomics.
//
// The blocks of the cluster meet at cluster barriers only (every block passes all of them, there is no wait that could run out). What they
// tell each other is in shared memory of all of them (a few sums) or in the caller's outputs.
//
// What bounds it: the first kernel a chain of trips to memory with a barrier behind each, the second the bytes of the copied pages. us: 12 sequences of 700
// positions go on, 8.0; 256 of 320 in 6,000 pages, 14.0; a pool of 701 pages compacted 10.5, one of 7,001 in 112 planes of 2 KB pages 130.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/sslm_b200.h"
#include "sslm_cluster.cuh"
#include "sslm_kernels.h"

namespace sslm {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMostSequences = 65535, kMostTable = 65536;
constexpr int kMostRange = 4096;      // sequences of a block: kMostSequences over 16 blocks
constexpr uint32_t kCopies = 0x80000000u, kRefused = 0xFFFFFFFFu;

// sums that every block has of every block
struct Told { alignas(8) uint32_t v[16][2]; };      // (a pair is stored as one word of 8 bytes)
__device__ __forceinline__ void tell(Told& told, int blocks, uint32_t a, uint32_t b) {      // (one thread per peer; a cluster barrier follows)
	static_assert(alignof(Told) == 8 && sizeof(told.v[0]) == 8, "a pair's place");
	if ((int)threadIdx.x < blocks) {
		const uint32_t at = cta_addr(told.v[cluster_rank()]);
		asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %1;\n\tst.shared::cluster.v2.u32 [ra], {%2, %3};\n\t}" ::"r"(at), "r"((uint32_t)threadIdx.x), "r"(a), "r"(b)
		             : "memory");
	}
}
__device__ __forceinline__ void meet() {
	__syncthreads();
	cluster_arrive();
	cluster_wait();
}
__device__ __forceinline__ uint32_t block_total(uint32_t v, uint32_t* s) {
	v = __reduce_add_sync(0xffffffffu, v);
	__syncthreads();
	if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
	__syncthreads();
	return __reduce_add_sync(0xffffffffu, (threadIdx.x & 31) < kWarps ? s[threadIdx.x & 31] : 0u);
}
// the sum of v over the threads in front of this one, and over all
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t* s, uint32_t* all) {
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	uint32_t upto = v;
#pragma unroll
	for (int o = 1; o < 32; o *= 2) {
		const uint32_t z = __shfl_up_sync(0xffffffffu, upto, o);
		if (lane >= o) upto += z;
	}
	__syncthreads();
	if (lane == 31) s[warp] = upto;
	__syncthreads();
	const uint32_t part = lane < kWarps ? s[lane] : 0u;
	*all = __reduce_add_sync(0xffffffffu, part);
	return upto - v + __reduce_add_sync(0xffffffffu, lane < warp ? part : 0u);
}
struct Range { int64_t from, to; };
__device__ __forceinline__ Range range_of(int64_t n, int blocks, int rank) {
	const int64_t each = (n + blocks - 1) / blocks;
	return Range{min(n, rank * each), min(n, (rank + 1) * each)};
}

__global__ void __launch_bounds__(kThreads) k_fork(const __grid_constant__ sslm_b200_fork a) {
	__shared__ Told s_told, s_free;
	__shared__ uint32_t s_part[kWarps], s_want[kMostRange];
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5, n = a.sequences, blocks = gridDim.x, rank = blockIdx.x;
	cluster_arrive();
	pdl_wait();
	pdl_release();
	cluster_wait();
	const Range seqs = range_of(n, blocks, rank), pages = range_of(a.num_pages, blocks, rank);
	const int first_held = pages.from + t < pages.to ? a.holders[pages.from + t] : 0;      // (asked for early; most ranges are a page a thread,
	auto held = [&](int64_t p) { return p == pages.from + t ? first_held : a.holders[p]; };
	// and a sequence a warp, whose record stays in registers)
	struct Seq { int parent, own, before, grow; } first{-1, 0, 0, 0};
	auto seq_of = [&](int64_t i) {
		Seq q{a.parents[i], a.lengths[i], 0, a.grow != nullptr ? a.grow[i] : 0};
		if (q.parent >= 0 && q.parent < n) q.before = q.parent == (int)i ? q.own : a.lengths[q.parent];
		return q;
	};
	const int room = a.table_pages * kPageTokens;
	auto used_of = [&](int length) { return length >= 0 && length <= room ? (length + kPageTokens - 1) / kPageTokens : 0; };
	// ---- what each sequence wants: a warp a sequence
	for (int64_t i = seqs.from + warp; i < seqs.to; i += kWarps) {
		const Seq q = seq_of(i);
		if (i == seqs.from + warp) first = q;
		const int parent = q.parent, before = q.before, grow = q.grow;
		int code = 0;
		uint32_t want = 0;
		if (parent < -1 || parent >= n) code = SSLM_B200_ROW_INDEX;
		else if (parent >= 0) {
			if (before < 0 || grow < 0 || before > room || grow > room - before) code = SSLM_B200_ROW_LENGTH;
			else {
				const bool moved = parent != (int)i;
				const int used = used_of(before), taken = moved ? before / kPageTokens : used;
				bool bad = false;
				if (moved)
					for (int j = lane; j < used; j += 32) {
						const int page = a.tables[parent * a.tables_stride + j];
						bad = bad || page < 0 || page >= a.num_pages;
					}
				if (__any_sync(0xffffffffu, bad)) code = SSLM_B200_ROW_INDEX;
				else want = (uint32_t)(used_of(before + grow) - taken) | (moved && before % kPageTokens != 0 ? kCopies : 0u);
			}
		}
		if (lane == 0) {
			a.status[i] = code;
			s_want[i - seqs.from] = code == 0 ? want : kRefused;
		}
	}
	// ---- free pages of this block's range
	uint32_t unheld = 0;
	for (int64_t p = pages.from + t; p < pages.to; p += kThreads) {
		const int h = held(p);
		a.out_holders[p] = h;
		unheld += h == 0 ? 1u : 0u;
	}
	__syncthreads();
	const int mine = (int)(seqs.to - seqs.from);
	uint32_t wanted = 0, copies = 0;
	for (int i = t; i < mine; i += kThreads) {
		const uint32_t want = s_want[i] == kRefused ? 0u : s_want[i];
		wanted += want & ~kCopies;
		copies += want >> 31;
	}
	wanted = block_total(wanted, s_part);
	copies = block_total(copies, s_part);
	unheld = block_total(unheld, s_part);
	tell(s_told, blocks, wanted, copies);
	tell(s_free, blocks, unheld, 0u);
	meet();
	uint32_t want_before = 0, copies_before = 0, free_before = 0, want_all = 0, free_all = 0;
	for (int i = 0; i < blocks; ++i) {
		if (i < rank) {
			want_before += s_told.v[i][0];
			copies_before += s_told.v[i][1];
			free_before += s_free.v[i][0];
		}
		want_all += s_told.v[i][0];
		free_all += s_free.v[i][0];
	}
	// ---- the pages that are drawn, in order
	const uint32_t last = min(want_all, free_all);
	for (int64_t p0 = pages.from; p0 < pages.to && free_before < last; p0 += kThreads) {
		const bool is_free = p0 + t < pages.to && held(p0 + t) == 0;
		uint32_t all;
		const uint32_t at = free_before + block_before(is_free ? 1u : 0u, s_part, &all);
		if (is_free && at < last) a.drawn[at] = (int32_t)(p0 + t);
		free_before += all;
	}
	meet();
	// ---- tables, lengths, holders and moves. First each sequence's place among the drawn pages and the moves, a thread a sequence
	uint32_t drawn = 0, moves = 0;
	for (int i0 = 0; i0 < mine; i0 += kThreads) {
		const int i = i0 + t;
		const bool refused = i < mine && s_want[i] == kRefused;
		const uint32_t want = i < mine && !refused ? s_want[i] : 0u;
		uint32_t all_want, all_copies;
		const uint32_t at = want_before + block_before(want & ~kCopies, s_part, &all_want), move = copies_before + block_before(want >> 31, s_part, &all_copies);
		want_before += all_want;
		copies_before += all_copies;
		if (i < mine) {
			const int64_t s = seqs.from + i;
			const uint32_t count = want & ~kCopies;
			const bool served = refused || count == 0u || (at <= free_all && count <= free_all - at);
			if (!served) a.status[s] = SSLM_B200_ROW_PAGES;
			else {
				drawn += count;
				if (want >> 31) {
					++moves;
					const int parent = a.parents[s];
					a.moves[2 * move] = a.tables[parent * a.tables_stride + a.lengths[parent] / kPageTokens];
					a.moves[2 * move + 1] = a.drawn[at];
				}
			}
			s_want[i] = served && !refused ? at : kRefused;      // (no place is that far back: the pages are fewer)
		}
	}
	__syncthreads();
	for (int64_t i = seqs.from + warp; i < seqs.to; i += kWarps) {
		const uint32_t at = s_want[i - seqs.from];
		const Seq q = i == seqs.from + warp ? first : seq_of(i);
		const int parent = q.parent, own_length = q.own;
		const int32_t* own = a.tables + i * a.tables_stride;
		int32_t* out = a.out_tables + i * a.out_stride;
		if (at == kRefused) {      // as it was
			for (int j = lane; j < used_of(own_length); j += 32) out[j] = own[j];
			if (lane == 0) a.out_lengths[i] = own_length;
			continue;
		}
		const bool moved = parent != (int)i;
		if (moved)      // what it held it lets go
			for (int j = lane; j < used_of(own_length); j += 32)
				if (own[j] >= 0 && own[j] < a.num_pages) atomicSub(&a.out_holders[own[j]], 1);
		int length = 0;
		if (parent >= 0) {
			const int before = q.before, taken = moved ? before / kPageTokens : used_of(before);
			length = before + q.grow;
			const int32_t* from = a.tables + parent * a.tables_stride;
			for (int j = lane; j < used_of(length); j += 32) {
				const int page = j < taken ? from[j] : a.drawn[at + (uint32_t)(j - taken)];
				out[j] = page;
				if (moved || j >= taken) atomicAdd(&a.out_holders[page], 1);
			}
		}
		if (lane == 0) a.out_lengths[i] = length;
	}
	drawn = block_total(drawn, s_part);
	moves = block_total(moves, s_part);
	tell(s_told, blocks, moves, drawn);
	meet();
	if (rank == 0 && t < 2) {
		uint32_t all = 0;
		for (int i = 0; i < blocks; ++i) all += s_told.v[i][t];
		a.counts[t] = (int32_t)all;
	}
}

__global__ void __launch_bounds__(kThreads) k_compact(const __grid_constant__ sslm_b200_compact a) {
	__shared__ Told s_told, s_moves;
	__shared__ uint32_t s_part[kWarps];
	const int t = threadIdx.x, lane = t & 31, warp = t >> 5, n = a.sequences, blocks = gridDim.x, rank = blockIdx.x;
	cluster_arrive();
	pdl_wait();
	pdl_release();
	cluster_wait();
	const Range pages = range_of(a.num_pages, blocks, rank);
	// (asked for early; most ranges are a page a thread, a sequence a warp, and a page of its table a lane)
	const int first_held = pages.from + t < pages.to ? a.holders[pages.from + t] : 0;
	auto held = [&](int64_t p) { return p == pages.from + t ? first_held : a.holders[p]; };
	const int64_t first_seq = (int64_t)rank * kWarps + warp;
	const int first_length = first_seq < n ? a.lengths[first_seq] : 0, first_page = first_seq < n && lane < a.table_pages ? a.tables[first_seq * a.tables_stride + lane] : -1;
	uint32_t used = 0;
	for (int64_t p = pages.from + t; p < pages.to; p += kThreads) used += held(p) != 0 ? 1u : 0u;
	used = block_total(used, s_part);
	tell(s_told, blocks, used, 0u);
	meet();
	int64_t live = 0;
	for (int i = 0; i < blocks; ++i) live += s_told.v[i][0];
	uint32_t holes = 0, late = 0;
	for (int64_t p = pages.from + t; p < pages.to; p += kThreads) {
		const int h = held(p);
		holes += h == 0 && p < live ? 1u : 0u;
		late += h != 0 && p >= live ? 1u : 0u;
		if (h == 0) a.new_of[p] = -1;
		else if (p < live) a.new_of[p] = (int32_t)p;
		if (h != 0 || p >= live) a.out_holders[p] = p < live ? h : 0;
	}
	holes = block_total(holes, s_part);
	late = block_total(late, s_part);
	tell(s_moves, blocks, holes, late);
	meet();
	uint32_t holes_before = 0, late_before = 0, moves = 0;
	for (int i = 0; i < blocks; ++i) {
		if (i < rank) {
			holes_before += s_moves.v[i][0];
			late_before += s_moves.v[i][1];
		}
		moves += s_moves.v[i][0];      // (as many holes as pages behind the front)
	}
	if (holes + late > 0)
		for (int64_t p0 = pages.from; p0 < pages.to; p0 += kThreads) {
			const int64_t p = p0 + t;
			const bool is_used = p < pages.to && held(p) != 0, hole = p < pages.to && p < live && !is_used, behind = is_used && p >= live;
			uint32_t all;      // (both sums in one: a tile has 512 pages)
			const uint32_t before = block_before((hole ? 1u : 0u) | (behind ? 1u << 16 : 0u), s_part, &all);
			if (hole) a.moves[2 * (int64_t)(holes_before + (before & 0xFFFFu)) + 1] = (int32_t)p;
			if (behind) a.moves[2 * (int64_t)(late_before + (before >> 16))] = (int32_t)p;
			holes_before += all & 0xFFFFu;
			late_before += all >> 16;
		}
	meet();
	int2 last{0, 0};      // (what the last one's page is held by is waited for behind the barrier)
	int last_held = 0;
	bool any = false;
	for (int64_t k = (int64_t)rank * kThreads + t; k < moves; k += (int64_t)blocks * kThreads) {
		if (any) a.out_holders[last.y] = last_held;
		last = *(const int2*)(a.moves + 2 * k);
		a.new_of[last.x] = last.y;
		last_held = a.holders[last.x];
		any = true;
	}
	if (rank == 0 && t == 0) {
		a.counts[0] = (int32_t)moves;
		a.counts[1] = (int32_t)live;
	}
	meet();
	if (any) a.out_holders[last.y] = last_held;
	const int room = a.table_pages * kPageTokens;
	for (int64_t i = first_seq; i < n; i += (int64_t)blocks * kWarps) {
		const int length = i == first_seq ? first_length : a.lengths[i], entries = length >= 0 && length <= room ? (length + kPageTokens - 1) / kPageTokens : 0;
		const int32_t* from = a.tables + i * a.tables_stride;
		int32_t* out = a.out_tables + i * a.out_stride;
		auto new_page = [&](int j) {
			const int page = i == first_seq && j == lane ? first_page : from[j];
			return page < 0 || page >= a.num_pages ? -1 : a.new_of[page];
		};
		const int page = lane < entries ? new_page(lane) : 0;
		bool bad = page < 0;
		for (int j = lane + 32; j < entries; j += 32) bad = bad || new_page(j) < 0;
		bad = __any_sync(0xffffffffu, bad);
		if (!bad) {
			if (lane < entries) out[lane] = page;
			for (int j = lane + 32; j < entries; j += 32) out[j] = new_page(j);
		}
		if (lane == 0 && a.status != nullptr) a.status[i] = length < 0 || length > room ? SSLM_B200_ROW_LENGTH : (bad ? SSLM_B200_ROW_INDEX : 0);
	}
}

// pages moves[k][0] -> moves[k][1] of every plane, counts[0] of them: a warp a page of a plane, 512 bytes a load and four loads at once.
// Four times the blocks that an SM holds: one that ends makes room for one whose loads are already on their way when the others store. 1,730
// pages of 2 KB in 112 planes, 0.79 GB read and written: 130 us, 6.1 TB/s; as many blocks as an SM holds 140, blocks of 64 to 256 threads 129 to
// 132, but their number costs small calls up to 10 us. The copied pages stay in the L2, the next attention reads them.
constexpr int kCopyThreads = 512, kCopyBlocks = 16;
__global__ void __launch_bounds__(kCopyThreads) k_copy_pages(int8_t* kv, int64_t num_pages, int planes, int page_bytes, const int32_t* moves, const int32_t* counts) {
	const int lane = threadIdx.x & 31;
	pdl_wait();
	pdl_release();
	const int64_t count = counts[0], items = count * planes, plane_bytes = num_pages * page_bytes;
	const int vectors = page_bytes >> 4;
	for (int64_t i = ((int64_t)blockIdx.x * kCopyThreads + threadIdx.x) >> 5; i < items; i += (int64_t)gridDim.x * (kCopyThreads / 32)) {
		const int64_t plane = i / count, k = i - plane * count;
		const int2 m = *(const int2*)(moves + 2 * k);
		const int4* from = (const int4*)(kv + plane * plane_bytes + (int64_t)m.x * page_bytes);
		int4* to = (int4*)(kv + plane * plane_bytes + (int64_t)m.y * page_bytes);
		for (int v = lane; v < vectors; v += 128) {
			int4 x[4];
#pragma unroll
			for (int u = 0; u < 4; ++u)
				if (v + 32 * u < vectors) x[u] = __ldcg(from + v + 32 * u);
#pragma unroll
			for (int u = 0; u < 4; ++u)
				if (v + 32 * u < vectors) to[v + 32 * u] = x[u];
		}
	}
}

template <typename A>
cudaError_t pages_launch(void (*kernel)(A), const A& a, int most_moves, cudaStream_t st) {
	// blocks of the cluster: one for every 512 pages, or 16 sequences
	int blocks = 1;
	while (blocks < 16 && (a.num_pages > (int64_t)blocks * kThreads || a.sequences > blocks * kWarps)) blocks *= 2;
	static PerDeviceOnce once;
	cudaError_t e = once_per_device(once, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); });
	if (e != cudaSuccess) return e;
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3(blocks);
	cfg.blockDim = dim3(kThreads);
	cfg.stream = st;
	cudaLaunchAttribute attr[2];
	attr[0].id = cudaLaunchAttributeClusterDimension;
	attr[0].val.clusterDim.x = (unsigned)blocks;
	attr[0].val.clusterDim.y = 1;
	attr[0].val.clusterDim.z = 1;
	attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[1].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = attr;
	cfg.numAttrs = pdl_enabled() ? 2 : 1;
	e = cudaLaunchKernelEx(&cfg, kernel, a);
	if (e != cudaSuccess || a.kv == nullptr || a.planes == 0 || most_moves == 0) return e;
	const int64_t items = (int64_t)most_moves * a.planes, each = kCopyThreads / 32;
	const int grid = (int)std::min<int64_t>((items + each - 1) / each, (int64_t)sm_count() * kCopyBlocks);
	return launch_pdl(k_copy_pages, dim3(grid), dim3(kCopyThreads), 0, st, a.kv, a.num_pages, (int)a.planes, (int)a.page_bytes, (const int32_t*)a.moves, (const int32_t*)a.counts);
}

// what the two calls have in common
template <typename A>
sslm_status pages_check(const A& c) {
	if (c.sequences < 0 || c.sequences > kMostSequences || c.table_pages < 0 || c.table_pages > kMostTable || c.num_pages < 0 || c.num_pages > 0x7FFFFFFF) return SSLM_INVALID_ARGUMENT;
	if (c.planes < 0 || c.reserved != 0 || c.tables_stride < c.table_pages || c.out_stride < c.table_pages) return SSLM_INVALID_ARGUMENT;
	if (c.kv && (c.page_bytes < 16 || (c.page_bytes & 15) != 0)) return SSLM_INVALID_ARGUMENT;
	return SSLM_OK;
}
template <typename... P>
bool words(P... p) { return ((((uintptr_t)p & 3) == 0) && ...); }
// memory that the runtime knows, or none
bool reachable(const void* p) {
	cudaPointerAttributes at;
	if (p == nullptr || (cudaPointerGetAttributes(&at, p) == cudaSuccess && at.type != cudaMemoryTypeUnregistered)) return true;
	cudaGetLastError();
	return false;
}

}  // namespace
}  // namespace sslm

using namespace sslm;

extern "C" sslm_status sslm_b200_fork_resident(const sslm_b200_fork* call, void* stream) {
	if (!call || call->struct_size != sizeof(sslm_b200_fork)) return SSLM_INVALID_ARGUMENT;
	const sslm_b200_fork& c = *call;
	const sslm_status st = pages_check(c);
	if (st != SSLM_OK) return st;
	const bool any = c.sequences > 0;
	if (!c.counts || (any && (!c.lengths || !c.parents || !c.out_lengths || !c.status || !c.moves))) return SSLM_INVALID_ARGUMENT;
	if (any && c.table_pages > 0 && (!c.tables || !c.out_tables)) return SSLM_INVALID_ARGUMENT;
	if (c.num_pages > 0 && (!c.holders || !c.out_holders || (any && !c.drawn))) return SSLM_INVALID_ARGUMENT;
	if (c.holders && c.holders == c.out_holders) return SSLM_INVALID_ARGUMENT;      // (read when others are written)
	if (any && ((c.tables && c.tables == c.out_tables) || c.lengths == c.out_lengths)) return SSLM_INVALID_ARGUMENT;
	if (!words(c.holders, c.tables, c.lengths, c.parents, c.grow, c.out_holders, c.out_tables, c.out_lengths, c.status, c.drawn, c.counts) || ((uintptr_t)c.moves & 7) ||
	    ((uintptr_t)c.kv & 15))
		return SSLM_MISALIGNED_BUFFER;
	// (no sequences: the holders are still to be handed on. A caller without sequences may have no cache either; such addresses are left alone)
	if (!any && (!reachable(c.holders) || !reachable(c.out_holders) || !reachable(c.counts))) return SSLM_OK;
	if (pages_launch(k_fork, c, c.sequences, (cudaStream_t)stream) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}

extern "C" sslm_status sslm_b200_compact_resident(const sslm_b200_compact* call, void* stream) {
	if (!call || call->struct_size != sizeof(sslm_b200_compact)) return SSLM_INVALID_ARGUMENT;
	const sslm_b200_compact& c = *call;
	const sslm_status st = pages_check(c);
	if (st != SSLM_OK) return st;
	if (!c.counts) return SSLM_INVALID_ARGUMENT;
	if (c.sequences > 0 && (!c.lengths || (c.table_pages > 0 && (!c.tables || !c.out_tables)))) return SSLM_INVALID_ARGUMENT;
	if (c.num_pages > 0 && (!c.holders || !c.out_holders || !c.new_of || (c.num_pages > 1 && !c.moves))) return SSLM_INVALID_ARGUMENT;
	if (c.holders && c.holders == c.out_holders) return SSLM_INVALID_ARGUMENT;
	if (c.sequences > 1 && c.table_pages > 0 && c.tables == c.out_tables && c.tables_stride != c.out_stride) return SSLM_INVALID_ARGUMENT;      // (a row would be another one's input)
	if (!words(c.holders, c.tables, c.lengths, c.out_holders, c.out_tables, c.new_of, c.counts, c.status) || ((uintptr_t)c.moves & 7) || ((uintptr_t)c.kv & 15))
		return SSLM_MISALIGNED_BUFFER;
	if (pages_launch(k_compact, c, (int)(c.num_pages / 2), (cudaStream_t)stream) != cudaSuccess) {
		cudaGetLastError();
		return SSLM_ALLOCATION_FAILED;
	}
	return SSLM_OK;
}
