// decay attention's scan on float32 (trl_decay_scan.h)
#include "trl_decay_scan.h"

namespace trl_decay {
void launch_f32(const Scans &all, int count, bool out, hipStream_t st) { launch<float>(all, count, out, st); }
}  // namespace trl_decay
