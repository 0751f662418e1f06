// Sequences of a 4-bit cache copied, forked, reordered and compacted: sequence i of a cache becomes sequence parents[i] of another one, or of
// itself.
#include "kv_device.hpp"

namespace mg {
namespace {

// What slot j of a sequence of L positions holds: position p of the source, `from` its slot there (-1: lost, zeros). False: no position.
struct GatherSlot {
    const KvCache& to;
    const KvCache& from;
    int len, from_len;
    __device__ __forceinline__ bool find(int j, int& slot) const {
        const int ring = to.cap - to.sinks, last = len - 1, from_ring = from.cap - from.sinks;
        int p = j;
        if (j >= to.sinks) {
            if (last < to.sinks) return false;
            const int newest = kv_slot(last, to.sinks, ring), back = newest - j;
            p = last - (back + (back < 0 ? ring : 0));
            if (p < to.sinks) return false;
        }
        if (p > last) return false;
        slot = p < from_len && (p < from.sinks || p >= from_len - from_ring) ? kv_slot(p, from.sinks, from_ring) : -1;
        return true;
    }
};

// Another cache's: a workgroup a sequence, head and stretch of slots, a lane 16 bytes of codes of K and V; then the scales, a slot a lane.
template <int DH>
__global__ __launch_bounds__(256) void kv_gather_kernel(KvGatherArgs a) {
    constexpr int row = DH / 2, L16 = row / 16, NB = DH / 32;
    const int i = blockIdx.x / a.to.heads, h = blockIdx.x - i * a.to.heads, parent = a.parents[i];
    if (parent < 0 || parent >= a.from.n) return;
    const int len = min(max(a.lens[i], 0), kKvMaxPos);
    const GatherSlot g{a.to, a.from, len, a.from_lens ? min(max(a.from_lens[parent], 0), kKvMaxPos) : len};
    const size_t to = ((size_t)i * a.to.heads + h) * a.to.cap, from = ((size_t)parent * a.to.heads + h) * a.from.cap;
    const int slots = min(len, a.to.cap), step = gridDim.y * 256;
    for (int x = blockIdx.y * 256 + threadIdx.x; x < slots * L16; x += step) {
        const int j = x / L16, at = 16 * (x % L16);
        int slot;
        if (!g.find(j, slot)) continue;
        u32x4 k = {}, v = {};
        if (slot >= 0) {
            k = *(const u32x4*)(a.from.k + (from + slot) * row + at);
            v = *(const u32x4*)(a.from.v + (from + slot) * row + at);
        }
        *(u32x4*)(a.to.k + (to + j) * row + at) = k;
        *(u32x4*)(a.to.v + (to + j) * row + at) = v;
    }
    for (int j = blockIdx.y * 256 + threadIdx.x; j < slots; j += step) {
        int slot;
        if (!g.find(j, slot)) continue;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            a.to.ks[(to + j) * NB + b] = slot >= 0 ? a.from.ks[(from + slot) * NB + b] : 0;
            a.to.vs[(to + j) * NB + b] = slot >= 0 ? a.from.vs[(from + slot) * NB + b] : 0;
        }
    }
}

// In place: as if from a copy. What a sequence's place is to hold may be another's old rows and so on around, so a workgroup takes 16 bytes
// of a head's plane times some neighbours, of all sequences at once: it reads all that moves there into its lanes' registers, waits, and
// writes. Nobody else touches these bytes. A lane writes what it read.
constexpr int kLanes = 1024, kHold = 16;         // lanes a workgroup, 16-byte pieces a lane
constexpr int kInPlaceMax = kLanes * kHold;      // sequences

template <int RB>
__device__ __forceinline__ void gather_columns(const KvGatherArgs& a, uint8_t* plane, int h, const uint32_t* moves, int moved, int per_wg) {
    const size_t seq = (size_t)a.to.heads * a.to.cap * RB;
    uint8_t* base = plane + (size_t)h * a.to.cap * RB;
    const uint32_t columns = (uint32_t)((size_t)a.to.cap * RB / 16);
    int shift = 0;  // 2^shift columns at once
    while ((2 << shift) <= per_wg && ((size_t)moved << (shift + 1)) <= (size_t)kInPlaceMax) shift++;
    const int width = 1 << shift, items = moved << shift;
    for (uint32_t c0 = blockIdx.x * per_wg; c0 < columns; c0 += gridDim.x * per_wg) {
        for (uint32_t c1 = c0; c1 < min(columns, c0 + per_wg); c1 += width) {
            u32x4 x[kHold];
            uint32_t fine = 0;
#pragma unroll
            for (int k = 0; k < kHold; k++) {
                const int n = k * kLanes + threadIdx.x;
                if (k * kLanes >= items) break;
                if (n >= items) continue;
                const uint32_t mv = moves[n >> shift], c = c1 + (n & (width - 1)), j = 16 * c / RB;
                const int i = mv >> 16, parent = mv & 0xffff;
                if (c >= columns || (int)j >= min(max(a.lens[i], 0), a.to.cap)) continue;
                fine |= 1u << k;
                x[k] = *(const u32x4*)(base + parent * seq + 16 * (size_t)c);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kHold; k++) {
                if (!(fine >> k & 1)) continue;
                const int n = k * kLanes + threadIdx.x;
                const uint32_t mv = moves[n >> shift], c = c1 + (n & (width - 1));
                const int i = mv >> 16, parent = mv & 0xffff, len = min(max(a.lens[i], 0), kKvMaxPos);
                uint8_t* to = base + i * seq + 16 * (size_t)c;
                const GatherSlot g{a.to, a.to, len, a.from_lens ? min(max(a.from_lens[parent], 0), kKvMaxPos) : len};
                if (!a.from_lens && (int)((16 * c + 15) / RB) < min(len, a.to.cap)) {
                    *(u32x4*)to = x[k];
                } else {
#pragma unroll
                    for (int b = 0; b < 16; b++) {
                        const int j = (16 * c + b) / RB;
                        int slot;
                        if (j < a.to.cap && g.find(j, slot)) to[b] = slot >= 0 ? (uint8_t)(x[k][b / 4] >> (8 * (b & 3))) : 0;
                    }
                }
            }
            __syncthreads();
        }
    }
}

template <int DH>
__global__ __launch_bounds__(kLanes) void kv_gather_in_place_kernel(KvGatherArgs a, int per_wg) {
    extern __shared__ uint32_t moves[];  // sequence << 16 | parent
    __shared__ int s_count[kLanes / 64];
    int moved = 0;
    for (int i0 = 0; i0 < a.to.n; i0 += kLanes) {
        const int i = i0 + threadIdx.x, parent = i < a.to.n ? a.parents[i] : -1;
        // (a sequence that becomes itself, of another length, may have positions to clear)
        const bool mv = parent >= 0 && parent < a.to.n && a.lens[i] > 0 && (parent != i || (a.from_lens && a.from_lens[i] != a.lens[i]));
        const uint64_t who = __ballot(mv);
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s_count[wave] = __popcll(who);
        __syncthreads();
        int before = moved;
        for (int w = 0; w < kLanes / 64; w++) {
            before += w < wave ? s_count[w] : 0;
            moved += s_count[w];
        }
        if (mv) moves[before + __popcll(who & ((1ull << (threadIdx.x & 63)) - 1))] = (uint32_t)i << 16 | parent;
    }
    __syncthreads();
    if (moved == 0) return;
    const int h = blockIdx.y >> 2;
    switch (blockIdx.y & 3) {
        case 0: return gather_columns<DH / 2>(a, a.to.k, h, moves, moved, per_wg);
        case 1: return gather_columns<DH / 2>(a, a.to.v, h, moves, moved, per_wg);
        case 2: return gather_columns<DH / 32>(a, a.to.ks, h, moves, moved, per_wg);
        default: return gather_columns<DH / 32>(a, a.to.vs, h, moves, moved, per_wg);
    }
}

bool in_place(const KvGatherArgs& a) { return a.to.k == a.from.k; }

}  // namespace

bool kv_gather_fits(const KvGatherArgs& a) {
    return in_place(a) ? a.to.n <= kInPlaceMax : (long long)a.to.n * a.to.heads < 1 << 23;
}

hipError_t launch_kv_gather(const KvGatherArgs& a, hipStream_t s) {
    return by_width(a.to.dh, [&](auto w) {
        constexpr int DH = decltype(w)::value;
        if (in_place(a)) {
            const int per_wg = 64;
            const long long blocks = ((long long)a.to.cap * (DH / 2) / 16 + per_wg - 1) / per_wg;
            const dim3 grid((unsigned)std::min<long long>(blocks, std::max(1, (1 << 16) / a.to.heads)), a.to.heads * 4);
            hipLaunchKernelGGL((kv_gather_in_place_kernel<DH>), grid, dim3(kLanes), 4 * a.to.n, s, a, per_wg);
            return hipGetLastError();
        }
        const long long rows = (long long)a.to.n * a.to.heads;
        const int blocks = (int)std::max<long long>(1, std::min<long long>((a.to.cap * (DH / 32) + 255) / 256, 8192 / rows));
        hipLaunchKernelGGL((kv_gather_kernel<DH>), dim3((unsigned)rows, blocks), dim3(256), 0, s, a);
        return hipGetLastError();
    });
}

}  // namespace mg
