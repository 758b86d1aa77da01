// attend_f32.hip - the attention kernels of attend.hpp for f32 caches (one
// type a file: they compile side by side).
#include "attend.hpp"

namespace aotk {

template void att_launch_kind<AOTK_F32>(int, int, int, const AttendLaunch &, uint32_t, hipStream_t);
template void att_join_kind<AOTK_F32>(int, const AttendLaunch &, uint32_t, uint32_t, uint32_t, uint64_t, uint32_t, hipStream_t);

}  // namespace aotk
