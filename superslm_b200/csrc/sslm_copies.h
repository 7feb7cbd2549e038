// The account of a block's bulk copies: chunks of data, numbered through all the block does, that take the places of a ring in
// turn, each place with a barrier that turns over once a chunk.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define SSLM_COPIES_FN __host__ __device__ __forceinline__
#else
#define SSLM_COPIES_FN inline
#endif

namespace sslm {

struct CopyAccount {
	uint32_t places;
	uint32_t issued;      // chunks asked for so far, in order

	SSLM_COPIES_FN uint32_t place(uint32_t chunk) const { return chunk % places; }
	SSLM_COPIES_FN uint32_t parity(uint32_t chunk) const { return chunk / places & 1u; }
	// a pass of `chunks` chunks begins behind `before` others, all of which have been used: how many are asked for at once
	SSLM_COPIES_FN uint32_t begin(uint32_t before, uint32_t chunks) {
		const uint32_t n = chunks < places ? chunks : places;
		issued = before + n;
		return n;
	}
	// chunk i of the pass has been used: whether another one takes its place. None does once a wait has run out.
	SSLM_COPIES_FN bool follows(uint32_t i, uint32_t chunks, bool late) {
		const bool more = !late && i + places < chunks;
		issued += more ? 1u : 0u;
		return more;
	}
	// the first of the chunks up to `issued` that may still be on their way: the last one of every place
	SSLM_COPIES_FN uint32_t open() const { return issued > places ? issued - places : 0u; }
};

}  // namespace sslm
