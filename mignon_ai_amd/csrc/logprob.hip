// Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits.
//
// With m the largest logit of a row, S = sum 2^((x - m) log2 e) and X = sum (x - m) of the same powers: log p(t) = x_t - m - log S, and
// the entropy is log S - X / S.
#include "logprob.hpp"

#include <algorithm>

#include "common.hpp"
#include "mx4_device.hpp"

namespace mg {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A logit and its place as one number: larger is likelier, the lowest id first among equals, -0 as 0, NaN below all.
__device__ __forceinline__ uint64_t top_key(float x, int id) {
    const uint32_t b = __float_as_uint(x + 0.0f), o = x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)o << 32 | (uint32_t)~id;
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor((unsigned long long)v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}

template <class T>
__global__ __launch_bounds__(256) void logprob_kernel(LogprobArgs a) {
    __shared__ float s_m[4], s_s[4], s_x[4];
    __shared__ uint64_t s_key[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (long long r = blockIdx.x; r < a.n; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.ld;
        float m = -INFINITY;
        bool nan = false;
        for (int v = threadIdx.x; v < a.V; v += 256) m = fmaxf(m, (float)x[v]);
        m = wave_max(m);
        __syncthreads();
        if (lane == 0) s_m[wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
        float S = 0.0f, X = 0.0f;
        for (int v = threadIdx.x; v < a.V; v += 256) {
            const float y = (float)x[v];
            const float far = y - m, e = __builtin_amdgcn_exp2f(far * kLog2e);
            S += e;
            X += e == 0.0f ? 0.0f : e * far;
        }
        S = wave_sum(S);
        X = wave_sum(X);
        if (lane == 0) {
            s_s[wave] = S;
            s_x[wave] = X;
        }
        __syncthreads();
        S = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
        X = (s_x[0] + s_x[1]) + (s_x[2] + s_x[3]);
        const float log_s = logf(S);
        if (a.entropy && threadIdx.x == 0) a.entropy[r] = log_s - X / S;
        for (int j = threadIdx.x; j < a.m; j += 256) {
            const int t = a.targets[r * a.m + j];
            a.logprob[r * a.m + j] = t >= 0 && t < a.V ? ((float)x[t] - m) - log_s : NAN;
        }
        uint64_t below = ~0ull;
        for (int j = 0; j < a.k; j++) {
            uint64_t best = 0;
            for (int v = threadIdx.x; v < a.V; v += 256) {
                const uint64_t key = top_key((float)x[v], v);
                if (key < below && key > best) best = key;
            }
            best = wave_max64(best);
            __syncthreads();
            if (lane == 0) s_key[wave] = best;
            __syncthreads();
            best = s_key[0];
            for (int w = 1; w < 4; w++) best = s_key[w] > best ? s_key[w] : best;
            below = best;
            if (threadIdx.x == 0) {
                const int id = (int)~(uint32_t)best;
                if (a.top_ids) a.top_ids[r * a.k + j] = id;
                if (a.top_logprob) a.top_logprob[r * a.k + j] = ((float)x[id] - m) - log_s;
            }
        }
    }
}

}  // namespace

size_t logprob_ws_bytes(const LogprobArgs& a) { return 0; }

hipError_t launch_logprob(const LogprobArgs& a, hipStream_t s) {
    return by_real(a.type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL((logprob_kernel<T>), dim3(std::min(a.n, 1 << 20)), dim3(256), 0, s, a);
        return hipGetLastError();
    });
}

}  // namespace mg
