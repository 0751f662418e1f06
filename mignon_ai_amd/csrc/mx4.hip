// Microscaled 4-bit rows: quantisation, reading back, and the product of two 4-bit matrices.
#include "mx4.hpp"

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "common.hpp"
#include "mx4_device.hpp"

namespace mg {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t Any16 __attribute__((ext_vector_type(4), may_alias));  // sixteen bytes of any type

// ---- Quantisation and reading back ----
// A workgroup of 256 lanes covers 256 / LC rows by 8 LC columns (LC lanes a row, four to a block, eight elements each): a lane
// reads 16 or 32 bytes and a wave writes whole lines of codes; the block's largest magnitude takes two exchanges among four
// lanes, so an element is read once and kept in registers. Bound by memory: 16384 x 4096 bf16, 170 MB each way, 35 us quantised
// (4.8 TB/s) and 26 read back (6.5), where a large copy reaches 4.9; 16 x 384 fp32 2.2 and 2.3 us, a launch.
constexpr int kRowLanes = 256;
constexpr int kMaxGridY = 32768;

template <class T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(Mx4RowsArgs a, int lc_log2) {
    const int lanes = ((a.K + 127) / 128) * 16;  // lanes a row
    const int rows = kRowLanes >> lc_log2;
    const int row_in = threadIdx.x >> lc_log2, c_in = threadIdx.x & ((1 << lc_log2) - 1);
    for (long long m = (long long)blockIdx.x * rows + row_in; m < a.M; m += (long long)gridDim.x * rows) {
        for (int c = (blockIdx.y << lc_log2) + c_in; c < lanes; c += gridDim.y << lc_log2) {
            float x[8];
            real_load8<T>((const T*)a.x + m * a.ld + 8 * c, a.K - 8 * c, x);
            uint32_t s;
            const uint32_t w = mx4_block(x, s);
            *(uint32_t*)(a.codes + m * lanes * 4 + 4 * c) = w;
            if ((c & 3) == 0) a.scales[m * (lanes >> 2) + (c >> 2)] = (uint8_t)s;
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(Mx4RowsArgs a, int lc_log2) {
    const int lanes = ((a.K + 127) / 128) * 16;
    const int rows = kRowLanes >> lc_log2;
    const int row_in = threadIdx.x >> lc_log2, c_in = threadIdx.x & ((1 << lc_log2) - 1);
    for (long long m = (long long)blockIdx.x * rows + row_in; m < a.M; m += (long long)gridDim.x * rows) {
        for (int c = (blockIdx.y << lc_log2) + c_in; 8 * c < a.K; c += gridDim.y << lc_log2) {
            float x[8];
            mx4_unpack8(*(const uint32_t*)(a.codes + m * lanes * 4 + 4 * c), mx4_scale(a.scales[m * (lanes >> 2) + (c >> 2)]), x);
            real_store8<T>((T*)a.y + m * a.ld + 8 * c, a.K - 8 * c, x);
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
// One 16-byte load per lane from global memory straight into LDS: lane L's bytes land at LDS offset lds + 16 L (four bytes: lds +
// 4 L). Inline assembly, with the waits written out (vm_wait), because the compiler would wait for all such loads before any LDS
// read. The LDS address goes through M0; the s_nop covers the wait states between a vector instruction's write of the scalar base
// and its use, and those of M0. No register receives anything.
__device__ __forceinline__ void lds_load16(const uint8_t* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "m0", "memory");
}
__device__ __forceinline__ void lds_load4(const uint8_t* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds) : "m0", "memory");
}
template <int N>
__device__ __forceinline__ void vm_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

// A workgroup of up to NW waves computes 16 FN channels x 16 FM rows, each wave over its own share of K, and adds the waves' sums in
// LDS, in the waves' order: for products with too few tiles to fill the chip, whose time is the latency of a tile's steps
// (1 x 384 by 8192 channels 2.8 us, of which the steps are one round trip to memory; 8 x 4096 by 4096 3.5). A
// wave's shares are runs of four steps; it loads them into four LDS slots of its own, which no other wave touches (no
// barriers), and reloads a slot once its products were issued. Slots and scales as in the large form.
template <int FN_, int FM_, int NW_>
struct MxSplit {
    static constexpr int FN = FN_, FM = FM_, NW = NW_, F = FN + FM;
    static constexpr int wave_lds = 4 * F * 1024 + 2 * F * 256, lds = NW * wave_lds;
    static_assert(4 * F <= 63 && lds <= 160 * 1024, "");
};

template <class S, class T>
__global__ __launch_bounds__(S::NW * 64) void mx4_gemm_split_kernel(Mx4GemmArgs a) {
    extern __shared__ uint8_t smem[];
    constexpr int FN = S::FN, FM = S::FM, F = S::F;
    const int L = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int n0 = blockIdx.x * 16 * FN, m0 = blockIdx.y * 16 * FM;
    const int steps = a.Kp / 128;
    const long long row = a.Kp / 2, srow = a.Kp / 32;
    const uint8_t* cb[F];
    const uint8_t* sb[F];
    uint32_t co[F], so[F];
#pragma unroll
    for (int f = 0; f < F; f++) {
        const bool w = f < FN;
        const int first = w ? n0 + 16 * f : m0 + 16 * (f - FN), last = (w ? a.N : a.M) - 1;
        const int r0 = min(first, last), r = min(first + (L >> 2), last) - r0;
        cb[f] = (w ? a.W : a.A) + r0 * row;
        co[f] = (uint32_t)(r * row) + 16 * ((L & 3) ^ ((L >> 3) & 3));
        sb[f] = (w ? a.Ws : a.As) + r0 * srow;
        so[f] = (uint32_t)(r * srow);
    }
    uint8_t* mine = smem + wave * S::wave_lds;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)mine;
    auto fetch = [&](int k) {
        const long long at = 64LL * min(k, steps - 1);
#pragma unroll
        for (int f = 0; f < F; f++) lds_load16(cb[f] + at, co[f], lds0 + ((k & 3) * F + f) * 1024);
    };
    auto fetch_scales = [&](int c, int slot) {
        const uint32_t at = 4 * min(4 * c + (L & 3), steps - 1);
#pragma unroll
        for (int f = 0; f < F; f++) lds_load4(sb[f], so[f] + at, lds0 + 4 * F * 1024 + (slot * F + f) * 256);
    };
    const int lane_at = (L & 15) * 64 + (((L >> 4) ^ ((L >> 1) & 3)) << 4);
    const uint32_t pick = (L >> 4) | (((L >> 4) + 4) << 8) | 0x0c0c0000u;
    v4f acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    int sc[F];
    auto step = [&](auto ss, auto more, int c, int next) {
        constexpr int s = decltype(ss)::value;
        constexpr bool MORE = decltype(more)::value;
        // the loads issued after this step's: three steps', and the next scales
        vm_wait<MORE ? 4 * F : (3 - s) * F>();
        if (4 * c + s < steps) {
            uint4 q[F];
#pragma unroll
            for (int f = 0; f < F; f++) q[f] = *(const uint4*)(mine + (s * F + f) * 1024 + lane_at);
#pragma unroll
            for (int i = 0; i < FN; i++) {
                const v8i w = {(int)q[i].x, (int)q[i].y, (int)q[i].z, (int)q[i].w, 0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < FM; j++) {
                    const uint4 p = q[FN + j];
                    const v8i x = {(int)p.x, (int)p.y, (int)p.z, (int)p.w, 0, 0, 0, 0};
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc[i][j], 4, 4, s, sc[i], s, sc[FN + j]);
                }
            }
        }
        if (MORE) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot's reads are done
            fetch(4 * next + s);
        }
    };
    auto run = [&](auto more, int c, int slot) {
        const int next = c + waves;
        if (decltype(more)::value) fetch_scales(next, slot ^ 1);
        vm_wait<(decltype(more)::value ? 5 : 4) * F>();  // this run's scales
#pragma unroll
        for (int f = 0; f < F; f++) {
            const uint4 q = *(const uint4*)(mine + 4 * F * 1024 + (slot * F + f) * 256 + (L & 15) * 16);
            sc[f] = (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(q.w, q.z, pick), __builtin_amdgcn_perm(q.y, q.x, pick), 0x05040100u);
        }
        step(std::integral_constant<int, 0>(), more, c, next);
        step(std::integral_constant<int, 1>(), more, c, next);
        step(std::integral_constant<int, 2>(), more, c, next);
        step(std::integral_constant<int, 3>(), more, c, next);
    };
    const int runs = (steps + 3) / 4;  // (at least as many as waves)
    fetch_scales(wave, 0);
    for (int s = 0; s < 4; s++) fetch(4 * wave + s);
    int c = wave, slot = 0;
    for (; c + waves < runs; c += waves, slot ^= 1) run(std::true_type(), c, slot);
    run(std::false_type(), c, slot);

    // the sums, fragment by fragment over the slots; wave w adds up fragments w, w + waves, ...
    __syncthreads();
    v4f* part = (v4f*)smem;
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++) part[(wave * FN * FM + i * FM + j) * 64 + L] = acc[i][j];
    __syncthreads();
    for (int f = wave; f < FN * FM; f += waves) {
        v4f sum = part[f * 64 + L];
        for (int w = 1; w < waves; w++) sum += part[(w * FN * FM + f) * 64 + L];
        const int i = f / FM, j = f - i * FM;
        const int m = m0 + 16 * j + (L & 15), n = n0 + 16 * i + 4 * (L >> 4);
        if (m < a.M) real_store4((T*)a.C + (long long)m * a.N + n, sum, a.N - n);
    }
}

// ---- Large products ----
// A workgroup of WN x WM waves computes TN channels x TM rows, each wave its FN x FM fragments of 16 x 16, in steps of 128
// elements of K. The codes of two steps, a line of 128 bytes a row, come into one of the LDS slots at once, those of the next
// pairs while a pair is worked on; the scales of four steps (16 bytes a row) into one of two. What the loads cost is lines
// touched, not bytes: eight neighbouring lanes take the line of a row. A fragment is 16 rows of 128 bytes in LDS, a row's eight
// blocks exchanged by row & 7 so that eight lanes reading one block of eight rows touch all banks. Two slots, or four where the
// tile is small and its steps are short.
//
// In a step each channel fragment is read anew for the next step right after its products were issued, so that only the row
// fragments need two sets of registers.
//
// 16384 x 4096 x 4096 into bf16: 154 us between other calls, 172 in a row of forty, where power holds the clock down (3.6 and 3.2
// PFLOP/s); 8192 x 8192 x 8192 303 us in such a row, 3.6: three times what a large bf16 product reaches on this card (1.26). The
// instruction alone, on random data in registers, reaches 5.8 to 6.4 (9 and more on zeros), which is 86 to 95 us for the products; the
// rest is what does not overlap with them: a tile's first loads and its output, which all workgroups write at about the same time
// (20 us at the rate of a fill). At the instruction's nominal rate a step of a 256 x 256 tile takes 1024 cycles of a CU's matrix units,
// and the step's LDS traffic (96 KiB read by the waves, 32 KiB written by the loads, 128 bytes a cycle) as many, so the tile is as
// large as registers allow (the table at gemm_tile has the smaller ones). Steps loaded one by one, 64 bytes a row, took 3 % longer,
// and an output of 32 bytes a row and store, straight from the registers, 8 %.
template <int TN_, int TM_, int WN_, int WM_, int SLOTS_>
struct MxTile {
    static constexpr int TN = TN_, TM = TM_, WN = WN_, WM = WM_, kSlots = SLOTS_;
    static constexpr int NW = WN * WM, FN = TN / 16 / WN, FM = TM / 16 / WM;
    static constexpr int loads = (TN + TM) / 16 / NW;  // of a wave: fragments whose codes and scales it loads
    static constexpr int slot = (TN + TM) * 128, o_scale = kSlots * slot, scale_slot = (TN + TM) * 16;
    static constexpr int ahead = kSlots == 2 ? 2 : kSlots - 1, o_out = o_scale + 2 * scale_slot, lds = o_out + NW * 2048;
    static_assert((TN + TM) / 16 % NW == 0 && FM <= FN && FN % 2 == 0 && (kSlots == 2 || kSlots == 4) && lds <= 160 * 1024, "");
};

template <class S, class T>
__global__ __launch_bounds__(S::NW * 64) void mx4_gemm_lds_kernel(Mx4GemmArgs a, int tiles_n, int tiles_m) {
    extern __shared__ uint8_t smem[];
    const int L = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave % S::WN, wm = wave / S::WN;
    // consecutive tiles stay on one XCD (its L2), in bands of eight channel tiles
    const int tile = xcd_tile(blockIdx.x, tiles_n * tiles_m);
    if (tile >= tiles_n * tiles_m) return;
    const int band = tile / (8 * tiles_m), in_band = tile - band * 8 * tiles_m;
    const int width = min(8, tiles_n - 8 * band);
    const int n0 = (8 * band + in_band % width) * S::TN, m0 = in_band / width * S::TM;
    const int steps = a.Kp / 128, pairs = (steps + 1) / 2;
    const long long row = a.Kp / 2, srow = a.Kp / 32;

    // this wave's loads: 16 rows each, first of W, then of A (rows past the end: the last one, whose results are not stored)
    const uint8_t* cb[S::loads];
    const uint8_t* sb[S::loads];
    uint32_t co[S::loads][2], so[S::loads];
    const uint32_t block = (L & 7) ^ (L >> 3), tail = 16 * (block & 4);
#pragma unroll
    for (int j = 0; j < S::loads; j++) {
        const int f = wave * S::loads + j;
        const bool w = f < S::TN / 16;
        const int first = w ? n0 + 16 * f : m0 + 16 * (f - S::TN / 16), last = (w ? a.N : a.M) - 1;
        const int r0 = min(first, last);
        cb[j] = (w ? a.W : a.A) + r0 * row;
        sb[j] = (w ? a.Ws : a.As) + r0 * srow;
#pragma unroll
        for (int h = 0; h < 2; h++) co[j][h] = (uint32_t)((min(first + 8 * h + (L >> 3), last) - r0) * row) + 16 * block;
        so[j] = (uint32_t)((min(first + (L >> 2), last) - r0) * srow);
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)smem + wave * S::loads * 2048;
    const uint32_t lds1 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)smem + S::o_scale + wave * S::loads * 256;
    // Past the last pair it is loaded again: the count of loads in flight stays the same. Of a pair with one step that one is loaded
    // twice.
    auto fetch = [&](int p, int slot) {
        const int q = min(p, pairs - 1);
        const uint32_t cut = 2 * q + 1 < steps ? 0 : tail;
#pragma unroll
        for (int j = 0; j < S::loads; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) lds_load16(cb[j] + 128LL * q, co[j][h] - cut, lds0 + slot * S::slot + 2048 * j + 1024 * h);
    };
    auto fetch_scales = [&](int c, int slot) {
        const uint32_t at = 4 * min(4 * c + (L & 3), steps - 1);
#pragma unroll
        for (int j = 0; j < S::loads; j++) lds_load4(sb[j], so[j] + at, lds1 + slot * S::scale_slot + 256 * j);
    };
    // of the first step of a pair; of the second: ^ 64
    const int lane_at = (L & 15) * 128 + (((L >> 4) ^ (L & 7)) << 4);
    auto read_w = [&](int at, int i) { return *(const uint4*)(smem + at + (wn * S::FN + i) * 2048); };
    auto read_a = [&](int at, int j) { return *(const uint4*)(smem + at + (S::TN / 16 + wm * S::FM + j) * 2048); };
    // the scale bytes of a lane's block in four steps, one a byte (the instruction picks one)
    const uint32_t pick = (L >> 4) | (((L >> 4) + 4) << 8) | 0x0c0c0000u;
    auto read_scale = [&](int slot, int r) {
        const uint4 q = *(const uint4*)(smem + S::o_scale + slot * S::scale_slot + (r + (L & 15)) * 16);
        return (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(q.w, q.z, pick), __builtin_amdgcn_perm(q.y, q.x, pick), 0x05040100u);
    };
    v4f acc[S::FN][S::FM];
#pragma unroll
    for (int i = 0; i < S::FN; i++)
#pragma unroll
        for (int j = 0; j < S::FM; j++) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    uint4 wf[S::FN], af[2][S::FM];
    int ws[S::FN], as[S::FM];
    auto scales = [&](int slot) {
#pragma unroll
        for (int i = 0; i < S::FN; i++) ws[i] = read_scale(slot, (wn * S::FN + i) * 16);
#pragma unroll
        for (int j = 0; j < S::FM; j++) as[j] = read_scale(slot, S::TN + (wm * S::FM + j) * 16);
    };
    auto barrier = [&] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // Step k = 4 c + s. Its row fragments are in af[s & 1], its channel fragments in wf, those of step k + 1 are read from LDS. The
    // second step of a pair waits until the next pair has landed (and scales that were asked for before it) and until every wave has
    // read this one, and loads a slot anew.
    auto step = [&](auto sc, int c) {
        constexpr int s = decltype(sc)::value;
        const int pair = 2 * c + (s >> 1);
        if (s & 1) {
            // (with more slots than two the one loaded anew was read in the pair before)
            if (S::kSlots == 2) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            vm_wait<2 * (S::ahead - 2) * S::loads>();
            barrier();
            if (s == 1) fetch_scales(c + 1, (c + 1) & 1);
            fetch(pair + S::ahead, (pair + S::ahead) % S::kSlots);
        }
        const int at = (lane_at ^ (s & 1 ? 0 : 64)) + (pair + (s & 1)) % S::kSlots * S::slot;
#pragma unroll
        for (int i = 0; i < S::FN; i++) {
            const v8i w = {(int)wf[i].x, (int)wf[i].y, (int)wf[i].z, (int)wf[i].w, 0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < S::FM; j++) {
                const uint4 q = af[s & 1][j];
                const v8i x = {(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc[i][j], 4, 4, s, ws[i], s, as[j]);
            }
            if (i < S::FM) af[(s + 1) & 1][i] = read_a(at, i);
            wf[i] = read_w(at, i);
            __builtin_amdgcn_sched_group_barrier(0x008, S::FM, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            if (i < S::FM) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (s == 3) scales((c + 1) & 1);
    };
    fetch_scales(0, 0);
    for (int p = 0; p < S::ahead; p++) fetch(p, p);
    vm_wait<2 * (S::ahead - 2) * S::loads>();
    barrier();
#pragma unroll
    for (int j = 0; j < S::FM; j++) af[0][j] = read_a(lane_at, j);
#pragma unroll
    for (int i = 0; i < S::FN; i++) wf[i] = read_w(lane_at, i);
    scales(0);
    const int whole = steps / 4, rest = steps - 4 * whole;
    for (int c = 0; c < whole; c++) {
        step(std::integral_constant<int, 0>(), c);
        step(std::integral_constant<int, 1>(), c);
        step(std::integral_constant<int, 2>(), c);
        step(std::integral_constant<int, 3>(), c);
    }
    if (rest > 0) step(std::integral_constant<int, 0>(), whole);
    if (rest > 1) step(std::integral_constant<int, 1>(), whole);
    if (rest > 2) step(std::integral_constant<int, 2>(), whole);
    vm_wait<0>();

    // Fragments leave through LDS, 16 rows of up to 128 bytes at a time, so that stores write whole lines. Lane L has row L & 15 and
    // four channels from 4 (L >> 4) of a fragment.
    uint8_t* mine = smem + S::o_out + wave * 2048;
    constexpr int group = std::min(S::FN, 128 / (16 * (int)sizeof(T)));  // fragments side by side
    constexpr int lanes = group * (int)sizeof(T), each = 16 / (int)sizeof(T);  // of a row, 16 bytes each
#pragma unroll
    for (int j = 0; j < S::FM; j++)
#pragma unroll
        for (int i0 = 0; i0 < S::FN; i0 += group) {
            const int m = m0 + (wm * S::FM + j) * 16, n = n0 + (wn * S::FN + i0) * 16;
#pragma unroll
            for (int i = 0; i < group; i++) {
                const int at = 4 * (int)sizeof(T) * (4 * i + (L >> 4)), r = L & 15;
                T v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = (T)acc[i0 + i][j][e];
                __builtin_memcpy(__builtin_assume_aligned(mine + r * 128 + (at ^ (16 * (r & 7))), sizeof(v)), v, sizeof(v));
            }
#pragma unroll
            for (int h = 0; h < lanes / 4; h++) {
                const int r = h * (64 / lanes) + L / lanes, x = L % lanes, left = a.N - n - x * each;
                const T* v = (const T*)(mine + r * 128 + 16 * (x ^ (r & 7)));
                T* out = (T*)a.C + (long long)(m + r) * a.N + n + x * each;
                if (m + r >= a.M) continue;
                if (left >= each) {
                    *(typename Raw16<sizeof(T)>::type*)out = *(const Any16*)v;
                } else {
                    for (int e = 0; e < left; e++) out[e] = v[e];
                }
            }
        }
}

template <class S, class T>
hipError_t launch_lds_gemm(const Mx4GemmArgs& a, hipStream_t s) {
    static std::atomic<uint64_t> allowed{0};
    if (const hipError_t e = allow_lds((const void*)mx4_gemm_lds_kernel<S, T>, S::lds, allowed); e != hipSuccess) return e;
    const int tn = (a.N + S::TN - 1) / S::TN, tm = (a.M + S::TM - 1) / S::TM;
    hipLaunchKernelGGL((mx4_gemm_lds_kernel<S, T>), dim3(xcd_grid(tn * tm)), dim3(S::NW * 64), S::lds, s, a, tn, tm);
    return hipGetLastError();
}

template <class S, class T>
hipError_t launch_split_gemm(const Mx4GemmArgs& a, hipStream_t s) {
    static std::atomic<uint64_t> allowed{0};
    if (const hipError_t e = allow_lds((const void*)mx4_gemm_split_kernel<S, T>, S::lds, allowed); e != hipSuccess) return e;
    const int waves = std::min(S::NW, (a.Kp / 128 + 3) / 4);
    const dim3 grid((a.N + 16 * S::FN - 1) / (16 * S::FN), (a.M + 16 * S::FM - 1) / (16 * S::FM));
    hipLaunchKernelGGL((mx4_gemm_split_kernel<S, T>), grid, dim3(64 * waves), waves * S::wave_lds, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx4_quantize(const Mx4RowsArgs& a, hipStream_t s) {
    if (a.M <= 0 || a.K <= 0) return hipErrorInvalidValue;
    const RowsGrid g = rows_grid(a.M, ((a.K + 127) / 128) * 16);
    return by_real(a.type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL((mx4_quantize_kernel<T>), g.grid, dim3(256), 0, s, a, g.lc_log2);
        return hipGetLastError();
    });
}

hipError_t launch_mx4_dequantize(const Mx4RowsArgs& a, hipStream_t s) {
    if (a.M <= 0 || a.K <= 0) return hipErrorInvalidValue;
    const RowsGrid g = rows_grid(a.M, ((a.K + 127) / 128) * 16);
    return by_real(a.type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL((mx4_dequantize_kernel<T>), g.grid, dim3(256), 0, s, a, g.lc_log2);
        return hipGetLastError();
    });
}

namespace {
// The largest tile of which there are enough for three quarters of the 256 CUs and which the shape fills to four fifths;
// where even those of 64 x 64 are too few (0), K is split. us at M x N x K into bf16, forty in a row, 256 / 128 / 64 tiles, split
// 32 x 32 and 16 x 16:
//   16384 x 4096 x 4096: 182 201 304;     3584 x 3584 x 4096: 35 43;    4096 x 2048 x 4096: 33 26;    4096 x 4096 x 384: 12.2 13.6 20.6
//   2048 x 2048 x 4096: 30 18.7 19.8 54;    1536 x 1024 x 2048: - 10.3 7.2;    1001 x 2048 x 1152: 12 7.9 6.3 10.8 14.9
//   256 x 4096 x 4096: 28 15.8 9.2 14.5 18.7;    128 x 4096 x 4096: 27 15.4 8.6 8.3 11.2;    300 x 300 x 8192: 49 27 13.4 5.9 6
//   8 x 4096 x 4096: 27 14.8 8.2 4.2 3.5;    16 x 8192 x 4096: 27 15.2 8.4 5 4.3
int gemm_tile(const Mx4GemmArgs& a) {
    if (a.M <= 16) return 0;
    for (const int tile : {256, 128, 64}) {
        const long long n = (a.N + tile - 1) / tile, m = ((long long)a.M + tile - 1) / tile;
        if (n * m >= 192 && (tile == 64 || 4.0 * n * m * tile * tile <= 5.0 * a.M * a.N)) return tile;
    }
    return 0;
}
}  // namespace

// A launch has fewer than 2^32 lanes (and whole eights of workgroups); a tile's rows past the last one have numbers, too.
bool mx4_gemm_fits(const Mx4GemmArgs& a) {
    const int tile = gemm_tile(a);
    if (!tile) return true;
    const long long n = (a.N + tile - 1) / tile, m = ((long long)a.M + tile - 1) / tile;
    return n * m <= (tile == 256 ? 1 << 23 : 1 << 24) - 8 && a.M < INT_MAX - 256;
}

hipError_t launch_mx4_gemm(const Mx4GemmArgs& a, hipStream_t s) {
    if (a.M <= 0 || a.N <= 0 || a.Kp <= 0 || a.Kp % 128 || !mx4_gemm_fits(a)) return hipErrorInvalidValue;
    return by_real(a.type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (a.M <= 16) return launch_split_gemm<MxSplit<1, 1, 8>, T>(a, s);
        switch (gemm_tile(a)) {
            case 256: return launch_lds_gemm<MxTile<256, 256, 2, 4, 2>, T>(a, s);
            case 128: return launch_lds_gemm<MxTile<128, 128, 2, 2, 2>, T>(a, s);
            case 64: return launch_lds_gemm<MxTile<64, 64, 2, 2, 4>, T>(a, s);
            default: return launch_split_gemm<MxSplit<2, 2, 8>, T>(a, s);
        }
    });
}

}  // namespace mg
