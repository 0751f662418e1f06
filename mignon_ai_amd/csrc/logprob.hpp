// Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits (logprob.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx4.hpp"  // RealType

namespace mg {

constexpr int kMaxTop = 64, kLogprobMaxV = 1 << 30, kLogprobMaxTargets = 1 << 30;  // (a lane counts in steps of 256: below 2^31)

struct LogprobArgs {
    const void* x = nullptr;           // logits [n][V], row stride ld elements
    int type = REAL_F32, n = 0, V = 0, m = 0, k = 0;
    long long ld = 0;
    const int32_t* targets = nullptr;  // [n][m]
    float* logprob = nullptr;          // [n][m]
    float* entropy = nullptr;          // [n]
    int32_t* top_ids = nullptr;        // [n][k]
    float* top_logprob = nullptr;      // [n][k]
    void* ws = nullptr;                // logprob_ws_bytes
};
size_t logprob_ws_bytes(const LogprobArgs& a);
bool logprob_fits(const LogprobArgs& a);  // a launch takes it
hipError_t launch_logprob(const LogprobArgs& a, hipStream_t s);

}  // namespace mg
