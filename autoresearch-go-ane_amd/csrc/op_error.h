// The per-thread message of the operators on caller-owned device buffers
// (ane_op_last_error), defined beside the classifier-head loss.
#pragma once

namespace ane {

int op_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

}  // namespace ane
