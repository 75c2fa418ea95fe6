// The error word of kernels with bounded waits: what gave up on one says so here, and its output is not valid.
// One word of pinned host memory for all GPUs of the process, so that reading it costs no copy: what a launch wrote
// is seen once its stream has been synchronised.  Codes: 501-515 and 599 fp8 products, 601-617 and 699 attention over
// drafted trees.
#pragma once

namespace nvb {

// Null where it cannot be had.
int* device_error_word();
// Its value (0: none; the last code wins), and with reset 0 from then on.
int device_error_code(int reset);

}  // namespace nvb
