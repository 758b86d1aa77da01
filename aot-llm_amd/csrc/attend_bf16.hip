// attend_bf16.hip - the attention kernels of attend.hpp for bf16 caches (one
// type a file: they compile side by side).
#include "attend.hpp"

namespace aotk {

template void att_launch_kind<AOTK_BF16>(int, int, int, const AttendLaunch &, uint32_t, hipStream_t);
template void att_join_kind<AOTK_BF16>(int, const AttendLaunch &, uint32_t, uint32_t, uint32_t, uint64_t, uint32_t, hipStream_t);

}  // namespace aotk
