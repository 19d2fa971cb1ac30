// Global norm of a list of tensors, and the list scaled to at most max_norm.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>
#include <vector>

namespace gradclip {

struct Item {            // one dense tensor; dtypes as in mx4_common.h
    const void* src;
    void* dst;           // where the scaled values go
    int64_t n;
    int src_dt, dst_dt;
};

enum Norm : int { L2 = 0, L1 = 1, LINF = 2 };

// doubles that a call wants
size_t workspace_doubles(const std::vector<Item>& items);

// norm[0] = the norm; work[0] = the factor min(1, max_norm / (norm + 1e-6)),
// where max_norm >= 0
void norm(const std::vector<Item>& items, int kind, double max_norm,
          float* norm, double* work, hipStream_t stream);

// dst = src * work[0], after norm()
void scale(const std::vector<Item>& items, const double* work,
           hipStream_t stream);

}  // namespace gradclip
