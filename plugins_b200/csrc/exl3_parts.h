// exl3_parts.h -- the counter of an item of work that is cut between CTAs: its low half counts the parts that have arrived, its
// high half those among them that brought nothing (their CTA gave up).  Zero between launches; the last part sees to that.
#pragma once
#include <cstdint>

#if defined(__CUDACC__)
#define EXL3_HD_PARTS __host__ __device__ __forceinline__
#else
#define EXL3_HD_PARTS inline
#endif

namespace exl3 {

constexpr int kMaxParts = 65535;

// What a part adds to the counter.
EXL3_HD_PARTS uint32_t part_arrival(bool brought) { return brought ? 1u : 0x10001u; }
// Whether all of an item's parts have arrived, and whether each brought what it had to.
EXL3_HD_PARTS bool parts_arrived(uint32_t counter, int parts) { return (counter & 0xFFFFu) == static_cast<uint32_t>(parts); }
EXL3_HD_PARTS bool parts_whole(uint32_t counter) { return counter >> 16 == 0u; }

}  // namespace exl3
