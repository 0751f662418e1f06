// Microscaled 4-bit rows: quantisation, reading back, and the product of two 4-bit matrices.
#include "mx4.hpp"

#include <algorithm>

#include "common.hpp"
#include "mx4_device.hpp"

namespace mg {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// A workgroup of 256 lanes covers 256 / LC rows by 8 LC columns (LC lanes a row, four to a block, eight elements each).
constexpr int kRowLanes = 256;
constexpr int kMaxGridY = 32768;

template <class T, bool VEC>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(Mx4RowsArgs a, int lc_log2) {
    const int lanes = ((a.K + 127) / 128) * 16;  // lanes a row
    const int rows = kRowLanes >> lc_log2;
    const int row_in = threadIdx.x >> lc_log2, c_in = threadIdx.x & ((1 << lc_log2) - 1);
    for (long long m = (long long)blockIdx.x * rows + row_in; m < a.M; m += (long long)gridDim.x * rows) {
        for (int c = (blockIdx.y << lc_log2) + c_in; c < lanes; c += gridDim.y << lc_log2) {
            float x[8];
            real_load8<T, VEC>((const T*)a.x + m * a.ld + 8 * c, a.K - 8 * c, x);
            uint32_t s;
            const uint32_t w = mx4_block(x, s);
            *(uint32_t*)(a.codes + m * lanes * 4 + 4 * c) = w;
            if ((c & 3) == 0) a.scales[m * (lanes >> 2) + (c >> 2)] = (uint8_t)s;
        }
    }
}

template <class T, bool VEC>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(Mx4RowsArgs a, int lc_log2) {
    const int lanes = ((a.K + 127) / 128) * 16;
    const int rows = kRowLanes >> lc_log2;
    const int row_in = threadIdx.x >> lc_log2, c_in = threadIdx.x & ((1 << lc_log2) - 1);
    for (long long m = (long long)blockIdx.x * rows + row_in; m < a.M; m += (long long)gridDim.x * rows) {
        for (int c = (blockIdx.y << lc_log2) + c_in; 8 * c < a.K; c += gridDim.y << lc_log2) {
            float x[8];
            mx4_unpack8(*(const uint32_t*)(a.codes + m * lanes * 4 + 4 * c), mx4_scale(a.scales[m * (lanes >> 2) + (c >> 2)]), x);
            real_store8<T, VEC>((T*)a.y + m * a.ld + 8 * c, a.K - 8 * c, x);
        }
    }
}

struct RowsGrid {
    dim3 grid;
    int lc_log2;
};
RowsGrid rows_grid(int M, int lanes) {
    int lc = 4;  // lanes is a multiple of 16
    while (lc < 8 && lanes % (2 << lc) == 0) lc++;
    const long long groups = ((long long)M + (kRowLanes >> lc) - 1) / (kRowLanes >> lc);
    return {dim3((unsigned)std::min<long long>(groups, 1 << 20), std::min((lanes >> lc), kMaxGridY)), lc};
}

// C = A W^T on v_mfma_scale_f32_16x16x128_f8f6f4. Both operands' rows are read in the instruction's layout: lane L holds row
// (L & 15) and block L >> 4 of a 128-element step, sixteen code bytes and one scale byte.
//
// A workgroup of `waves` waves computes 16 channels x 16 rows, each wave over its share of the steps, and adds the waves'
// sums in LDS, in the waves' order.
template <class T>
__global__ __launch_bounds__(512) void mx4_gemm_tile_kernel(Mx4GemmArgs a) {
    __shared__ v4f part[7][64];
    const int L = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int n0 = blockIdx.x * 16;
    const int steps = a.Kp / 128;
    for (int m0 = blockIdx.y * 16; m0 < a.M; m0 += gridDim.y * 16) {
        const long long wr = min(n0 + (L & 15), a.N - 1), ar = min(m0 + (L & 15), a.M - 1);
        const uint8_t* wp = a.W + wr * (a.Kp / 2) + 16 * (L >> 4);
        const uint8_t* ap = a.A + ar * (a.Kp / 2) + 16 * (L >> 4);
        const uint8_t* wsp = a.Ws + wr * (a.Kp / 32) + (L >> 4);
        const uint8_t* asp = a.As + ar * (a.Kp / 32) + (L >> 4);
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = wave; k < steps; k += waves) {
            const uint4 wq = *(const uint4*)(wp + 64LL * k), aq = *(const uint4*)(ap + 64LL * k);
            const int ws = wsp[4 * k], as = asp[4 * k];
            const v8i wv = {(int)wq.x, (int)wq.y, (int)wq.z, (int)wq.w, 0, 0, 0, 0};
            const v8i av = {(int)aq.x, (int)aq.y, (int)aq.z, (int)aq.w, 0, 0, 0, 0};
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, av, acc, 4, 4, 0, ws, 0, as);
        }
        if (wave) part[wave - 1][L] = acc;
        __syncthreads();
        if (wave == 0) {
            for (int w = 1; w < waves; w++) acc += part[w - 1][L];
            // lane L: row m0 + (L & 15), channels n0 + 4 (L >> 4) .. + 3
            const int m = m0 + (L & 15), n = n0 + 4 * (L >> 4);
            T* out = (T*)a.C + (long long)m * a.N + n;
            if (m < a.M)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (n + r < a.N) out[r] = (T)acc[r];
        }
        __syncthreads();
    }
}

}  // namespace

hipError_t launch_mx4_quantize(const Mx4RowsArgs& a, hipStream_t s) {
    if (a.M <= 0 || a.K <= 0) return hipErrorInvalidValue;
    const RowsGrid g = rows_grid(a.M, ((a.K + 127) / 128) * 16);
    const bool vec = (uintptr_t)a.x % 16 == 0 && a.ld * real_size(a.type) % 16 == 0;
    return by_real(a.type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (vec) hipLaunchKernelGGL((mx4_quantize_kernel<T, true>), g.grid, dim3(256), 0, s, a, g.lc_log2);
        else hipLaunchKernelGGL((mx4_quantize_kernel<T, false>), g.grid, dim3(256), 0, s, a, g.lc_log2);
        return hipGetLastError();
    });
}

hipError_t launch_mx4_dequantize(const Mx4RowsArgs& a, hipStream_t s) {
    if (a.M <= 0 || a.K <= 0) return hipErrorInvalidValue;
    const RowsGrid g = rows_grid(a.M, ((a.K + 127) / 128) * 16);
    const bool vec = (uintptr_t)a.y % 16 == 0 && a.ld * real_size(a.type) % 16 == 0;
    return by_real(a.type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (vec) hipLaunchKernelGGL((mx4_dequantize_kernel<T, true>), g.grid, dim3(256), 0, s, a, g.lc_log2);
        else hipLaunchKernelGGL((mx4_dequantize_kernel<T, false>), g.grid, dim3(256), 0, s, a, g.lc_log2);
        return hipGetLastError();
    });
}

hipError_t launch_mx4_gemm(const Mx4GemmArgs& a, hipStream_t s) {
    if (a.M <= 0 || a.N <= 0 || a.Kp <= 0 || a.Kp % 128) return hipErrorInvalidValue;
    const int waves = std::max(1, std::min(8, a.Kp / 128));
    const dim3 grid((a.N + 15) / 16, std::min((a.M + 15) / 16, kMaxGridY));
    return by_real(a.type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL((mx4_gemm_tile_kernel<T>), grid, dim3(64 * waves), 0, s, a);
        return hipGetLastError();
    });
}

}  // namespace mg
