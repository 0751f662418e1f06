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
// 64 sequences of 1500 to 3000 positions, 8 heads of 128, 131 MB read and written: 23 us where the source stays in the caches (5.7 TB/s), and
// 41 on other data each call, where a plain copy of as many bytes takes 26: a lane asks for one pair of pieces, waits, and stores it before the
// next, and scales go byte by byte.
template <int DH>
__global__ __launch_bounds__(256) void kv_gather_kernel(KvGatherArgs a) {
    constexpr int row = DH / 2, L16 = row / 16, NB = DH / 32;
    const int i = blockIdx.x / a.to.heads, h = blockIdx.x - i * a.to.heads, parent = a.parents[i];
    if (parent < 0 || parent >= a.from.n) return;
    const int len = min(max(a.lens[i], 0), kKvMaxPos);
    const GatherSlot g{a.to, a.from, len, a.from_lens ? min(max(a.from_lens[parent], 0), kKvMaxPos) : len};
    const size_t to = ((size_t)i * a.to.heads + h) * a.to.cap, from = ((size_t)parent * a.to.heads + h) * a.from.cap;
    const int slots = min(len, a.to.cap), step = gridDim.y * 256;
    for (long long x = blockIdx.y * 256 + threadIdx.x; x < (long long)slots * L16; x += step) {
        const int j = (int)(x / L16), at = 16 * (int)(x % L16);
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
    for (int j = blockIdx.y * 256 + threadIdx.x; j < slots; j += step) {  // (slots and a step stay below 2^31)
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
// of a head's plane, times some neighbours, of all sequences at once: it reads all that moves there into its lanes' registers, waits, and
// writes. Nobody else touches these bytes, and a lane writes what it read. No memory beside the cache, each byte moved once.
//
// A lane holds HOLD pieces of 16 bytes: up to 512 sequences 256 lanes of 8, up to 2048 512 of 8, up to 16384 1024 of 16, so that whole 64 bytes
// of a place are taken together. us, half of the sequences becoming copies of the others, 256 x 8, 512 x 8, 1024 x 8 and 1024 x 16: 64 of 1024
// positions (8 heads of 128) 11.3 14.1 16.5 17; 256 of 1051 (8 of 64) 22 26 29 34; 1024 of 251 (8 of 64) 46 35 33 41; 2000 of 251 (8 of 32)
// 53 44 49 62; 4096 of 59 (8 of 32) - 51 46 45. Few long sequences (256 streams of 1056 slots, half of them moving, 111 MB
// read and written) take 22 us, 5 TB/s, where they stay in the caches, and 35 on other data each call, where a plain copy of as many bytes takes
// 22: a workgroup asks for all it holds, 128 bytes of a place, waits, and only then writes. Many are bound by lines of which a workgroup takes
// a part, and by the list of moves that each makes (4096: four rounds).
constexpr int kInPlaceMax = 1024 * 16;  // sequences

// Bytes of a piece one by one: up to the first slot that holds no position, or where some may have been lost (zeros).
__device__ __forceinline__ uint8_t byte_of(const u32x4& v, uint32_t b) {
    const uint32_t w = b < 8 ? (b < 4 ? v.x : v.y) : b < 12 ? v.z : v.w;
    return (uint8_t)(w >> (8 * (b & 3)));
}
template <int RB>
__device__ __forceinline__ void store_first(uint8_t* to, const u32x4& v, uint64_t first, uint32_t slots) {
    const uint32_t n = (uint32_t)min((uint64_t)16, (uint64_t)slots * RB - first);
#pragma unroll 1
    for (uint32_t b = 0; b < n; b++) to[b] = byte_of(v, b);
}
template <int RB>
__device__ __forceinline__ void store_some(uint8_t* to, const u32x4& v, const GatherSlot& g, uint64_t first) {
#pragma unroll 1
    for (uint32_t b = 0; b < 16; b++) {
        int slot;
        if (g.find((int)((first + b) / RB), slot)) to[b] = slot >= 0 ? byte_of(v, b) : 0;
    }
}

template <int RB, int NT, int HOLD>
__device__ __forceinline__ void gather_columns(const KvGatherArgs& a, uint8_t* plane, int h, const uint2* moves, int moved, uint32_t c0, int per_wg) {
    const size_t seq = (size_t)a.to.heads * a.to.cap * RB;
    uint8_t* base = plane + (size_t)h * a.to.cap * RB;
    const uint32_t columns = (uint32_t)((size_t)a.to.cap * RB / 16), c_end = min(columns, c0 + per_wg);
    int shift = 0;  // 2^shift columns at once
    while ((2 << shift) <= per_wg && (moved << (shift + 1)) <= NT * HOLD) shift++;
    const int width = 1 << shift, items = moved << shift;
    for (uint64_t c1 = c0; c1 < c_end; c1 += width) {
        u32x4 x[HOLD];
        uint32_t fine = 0;
#pragma unroll
        for (int k = 0; k < HOLD; k++) {
            const int n = k * NT + threadIdx.x;
            if (n >= items) continue;
            const uint2 mv = moves[n >> shift];
            const uint64_t c = c1 + (n & (width - 1));
            if (c >= c_end || 16 * c / RB >= mv.y) continue;
            fine |= 1u << k;
            x[k] = *(const u32x4*)(base + (mv.x & 0xffff) * seq + 16 * c);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int k = 0; k < HOLD; k++) {
            if (!(fine >> k & 1)) continue;
            int n = k * NT + threadIdx.x;
            asm volatile("" : "+v"(n));  // (addresses are found again: kept, they would not fit the registers)
            const uint2 mv = moves[n >> shift];
            const uint64_t c = c1 + (n & (width - 1));
            const uint32_t i = mv.x >> 16, parent = mv.x & 0xffff;
            uint8_t* to = base + i * seq + 16 * c;
            if (!a.from_lens && (16 * c + 15) / RB < mv.y) {
                *(u32x4*)to = x[k];
            } else if (!a.from_lens) {
                store_first<RB>(to, x[k], 16 * c, mv.y);
            } else {
                store_some<RB>(to, x[k], GatherSlot{a.to, a.to, min(max(a.lens[i], 0), kKvMaxPos), min(max(a.from_lens[parent], 0), kKvMaxPos)}, 16 * c);
            }
        }
        __syncthreads();
    }
}

template <int DH, int NT, int HOLD>
__global__ __launch_bounds__(NT) void kv_gather_in_place_kernel(KvGatherArgs a, int per_wg, int code_blocks, int scale_blocks) {
    extern __shared__ uint2 moves[];  // sequence << 16 | parent; slots that hold a position
    __shared__ int s_count[NT / 64];
    int moved = 0;
    for (int i0 = 0; i0 < a.to.n; i0 += NT) {
        const int i = i0 + threadIdx.x, parent = i < a.to.n ? a.parents[i] : -1, len = i < a.to.n ? a.lens[i] : 0;
        // (a sequence that becomes itself, of another length, may have positions to clear)
        const bool mv = parent >= 0 && parent < a.to.n && len > 0 && (parent != i || (a.from_lens && a.from_lens[i] != len));
        const uint64_t who = __ballot(mv);
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s_count[wave] = __popcll(who);
        __syncthreads();
        int before = moved;
        for (int w = 0; w < NT / 64; w++) {
            before += w < wave ? s_count[w] : 0;
            moved += s_count[w];
        }
        if (mv) moves[before + __popcll(who & ((1ull << (threadIdx.x & 63)) - 1))] = make_uint2((uint32_t)i << 16 | parent, min(len, a.to.cap));
    }
    __syncthreads();
    if (moved == 0) return;
    int b = blockIdx.x;
    const int codes = 2 * a.to.heads * code_blocks;
    if (b < codes) {
        const int plane = b / code_blocks, h = plane >> 1;
        gather_columns<DH / 2, NT, HOLD>(a, plane & 1 ? a.to.v : a.to.k, h, moves, moved, (uint32_t)(b - plane * code_blocks) * per_wg, per_wg);
    } else {
        b -= codes;
        const int plane = b / scale_blocks, h = plane >> 1;
        gather_columns<DH / 32, NT, HOLD>(a, plane & 1 ? a.to.vs : a.to.ks, h, moves, moved, (uint32_t)(b - plane * scale_blocks) * per_wg, per_wg);
    }
}

bool in_place(const KvGatherArgs& a) { return a.to.k == a.from.k; }

int in_place_lanes(const KvGatherArgs& a) { return a.to.n <= 512 ? 256 : a.to.n <= 2048 ? 512 : 1024; }

// Columns of a workgroup: the first power of two, up to 256, of which all sequences together fill its room (fewer than all move).
struct InPlacePlan {
    int per_wg;
    long long code_blocks, scale_blocks, blocks;
};
InPlacePlan in_place_plan(const KvGatherArgs& a, int room) {
    InPlacePlan p;
    p.per_wg = 1;
    while (p.per_wg < 256 && p.per_wg * a.to.n < room) p.per_wg *= 2;
    const auto blocks = [&](int rb) { return ((long long)a.to.cap * rb / 16 + p.per_wg - 1) / p.per_wg; };
    p.code_blocks = blocks(a.to.dh / 2);
    p.scale_blocks = blocks(a.to.dh / 32);
    p.blocks = 2 * a.to.heads * (p.code_blocks + p.scale_blocks);
    return p;
}

template <int DH, int NT, int HOLD>
hipError_t launch_in_place(const KvGatherArgs& a, hipStream_t s) {
    static std::atomic<uint64_t> allowed{0};
    if (NT == 1024)
        if (const hipError_t e = allow_lds((const void*)kv_gather_in_place_kernel<DH, NT, HOLD>, 8 * kInPlaceMax, allowed); e != hipSuccess) return e;
    const InPlacePlan p = in_place_plan(a, NT * HOLD);
    hipLaunchKernelGGL((kv_gather_in_place_kernel<DH, NT, HOLD>), dim3((unsigned)p.blocks), dim3(NT), 8 * a.to.n, s, a, p.per_wg, (int)p.code_blocks,
                       (int)p.scale_blocks);
    return hipGetLastError();
}

}  // namespace

// (a launch's 2^32 lanes)
bool kv_gather_fits(const KvGatherArgs& a) {
    if (!in_place(a)) return (long long)a.to.n * a.to.heads < 1 << 23;
    const int lanes = in_place_lanes(a);
    return a.to.n <= kInPlaceMax && in_place_plan(a, lanes * (lanes == 1024 ? 16 : 8)).blocks < (1LL << 32) / lanes;
}

hipError_t launch_kv_gather(const KvGatherArgs& a, hipStream_t s) {
    return by_width(a.to.dh, [&](auto w) {
        constexpr int DH = decltype(w)::value;
        if (in_place(a)) {
            switch (in_place_lanes(a)) {
                case 256: return launch_in_place<DH, 256, 8>(a, s);
                case 512: return launch_in_place<DH, 512, 8>(a, s);
                default: return launch_in_place<DH, 1024, 16>(a, s);
            }
        }
        const long long rows = (long long)a.to.n * a.to.heads;
        const int blocks = (int)std::max<long long>(1, std::min(((long long)a.to.cap * (DH / 32) + 255) / 256, 8192 / rows));
        hipLaunchKernelGGL((kv_gather_kernel<DH>), dim3((unsigned)rows, blocks), dim3(256), 0, s, a);
        return hipGetLastError();
    });
}

}  // namespace mg
