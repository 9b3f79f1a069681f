// What a kernel that looks page numbers over says about one that is not there.
#pragma once

#include "common.cuh"

namespace b200 {

// What stands for the sequence where the table is that of a prefix which all sequences share.
constexpr int kSharedPrefix = -1;

// A position whose page is not there is reported once: the row's when writing, which is left out, the page's first when reading.
// Attention reads page 0 instead.
__device__ __forceinline__ void report_page(int* status, int error, int b, int pos, int n_pages) {
  if (status != nullptr && atomicCAS(status, 0, error) == 0) {
    status[1] = b;
    status[2] = pos;
    status[3] = n_pages;
  }
}

}  // namespace b200
