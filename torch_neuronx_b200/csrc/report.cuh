// What a kernel that looks page numbers over says about one that is not there.
#pragma once

#include "common.cuh"

namespace b200 {

// A position whose page is not there is reported once.  Its write is left out, its read takes page 0 instead.
__device__ __forceinline__ void report_page(int* status, int error, int b, int pos, int n_pages) {
  if (status != nullptr && atomicCAS(status, 0, error) == 0) {
    status[1] = b;
    status[2] = pos;
    status[3] = n_pages;
  }
}

}  // namespace b200
