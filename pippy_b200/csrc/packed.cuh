// Documents packed into rows: what the kernels of csrc/packed.cu leave in device memory for the attention kernels.
#pragma once
#include <cuda_runtime.h>

namespace pbk {

// A device error word value of this file's kernels (ops._lib.check_device_errors names it).
constexpr int ERR_LAYOUT = 6;  // document lengths that are negative or do not fit their row
constexpr int ERR_INDEX = 5;   // a position outside its table

// One tile of kRows consecutive rows of a document (or of the padding behind a row's last document).
struct __align__(16) Tile {
  int start;  // first row of the document in the batch of rows * tokens_per_row rows
  int len;    // rows of the document
  int rank;   // this tile is rows [rank * kRows, min(len, (rank + 1) * kRows)) of it
  int pad;    // 1: padding, the results are zeros
};

}  // namespace pbk
