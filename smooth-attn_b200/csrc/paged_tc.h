// Launch plan of the tensor-core paged-decode kernel (paged_tc.cu), shared
// with the entry point in paged.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace sa {

// The tickets come first in a workspace that calls of other shapes have used before, and
// must be found zero.  So much of it is theirs whatever the shape, and no partial record
// lies there; a call of more units than that holds (16384) clears its tickets itself.
constexpr int64_t kTicketReserve = 65536;
inline int64_t ticket_bytes_of(int64_t units) { return std::max(kTicketReserve, (units * 4 + 255) / 256 * 256); }

struct PtcPlan {
  int GT;                // query heads per unit (the MMA's N columns in use)
  int64_t grid;          // CTAs (one per SM at most)
  int slots;             // partial-record slots per unit
  int64_t ticket_bytes;  // tickets [units]: ticket_bytes_of(units)
  int64_t part_bytes;    // partial records [units][slots][GT*128 + 16] fp32
};

bool paged_tc_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t max_blocks, int64_t bs, int64_t D, int dtype,
                   int sms, PtcPlan* p);
int paged_tc_launch(const void* q, const void* k_cache, const void* v_cache, void* out, const int32_t* bt,
                    const int32_t* cl, void* workspace, int64_t B, int64_t Hq, int64_t Hkv, int64_t num_blocks,
                    int64_t bs, int64_t max_blocks, float scale, const PtcPlan& p, cudaStream_t st);

}  // namespace sa
