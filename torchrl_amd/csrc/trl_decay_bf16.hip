// decay attention's scan on bfloat16 (trl_decay_scan.h)
#include "trl_decay_scan.h"

namespace trl_decay {
void launch_bf16(const Scans &all, int count, bool out, hipStream_t st) { launch<trl_bf16>(all, count, out, st); }
}  // namespace trl_decay
