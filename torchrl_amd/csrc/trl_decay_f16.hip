// decay attention's scan on float16 (trl_decay_scan.h)
#include "trl_decay_scan.h"

namespace trl_decay {
void launch_f16(const Scans &all, int count, bool out, hipStream_t st) { launch<trl_f16>(all, count, out, st); }
}  // namespace trl_decay
