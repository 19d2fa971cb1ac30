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

// A list, laid out for its launches.
class List {
public:
    explicit List(const std::vector<Item>& items);
    ~List();
    List(const List&) = delete;
    List& operator=(const List&) = delete;

    // doubles that a call wants
    size_t workspace_doubles() const;
    // norm[0] = the norm
    void norm(int kind, float* norm, double* work, hipStream_t stream) const;
    // the same, and dst = src * min(1, max_norm / (norm + 1e-6)), max_norm >= 0
    void clip(int kind, double max_norm, float* norm, double* work,
              hipStream_t stream) const;

private:
    struct Data;
    Data* d;
    int sums(int kind, double* part, hipStream_t stream) const;
};

}  // namespace gradclip
