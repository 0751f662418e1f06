// A key/value cache in microscaled 4-bit blocks: rows quantised as they are written, read back, and attention over them with
// a sliding window and a few first positions (sinks) that stay visible.
#include "mx4.hpp"

#include <algorithm>
#include <climits>

#include "common.hpp"
#include "mx4_device.hpp"

namespace mg {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// What a sequence's call covers: token t < count sits at position pos + t, the cache holds positions below `end`.
struct SeqSpan {
    int pos, count, end;
};
__device__ __forceinline__ SeqSpan seq_span(const int32_t* pos, const int32_t* counts, int s, int T) {
    SeqSpan r;
    r.pos = pos ? min(max(pos[s], -kKvMaxPos), kKvMaxPos) : 0;
    r.count = counts ? min(max(counts[s], 0), T) : T;
    r.end = r.pos + r.count;
    return r;
}
__device__ __forceinline__ int kv_slot(int p, int sinks, int ring) { return p < sinks ? p : sinks + (p - sinks) % ring; }

// ---- writing and reading rows --------------------------------------------------------------------------------------
// One launch for keys and values (blockIdx.z), a workgroup for 256 / (DH / 8) tokens of U heads (blockIdx.y): DH / 8 lanes a row, four
// to a block, a lane's U rows loaded before the first is worked on. Tokens that follow each other fill whole lines of codes and
// scales, and a token's heads are read side by side (32768 tokens of 8 bf16 heads of 128 written: one head a
// workgroup 53 us, four 44; read back 28 and 27). Bound by memory: 16 prompts of 1 to 2048 such tokens, 55 MB each way, 16 us
// (3.5 TB/s) and 13 (4.2); a decode step's 4096 tokens of 8 fp32 heads of 32 take 4.9 and 5.3 us, the latency of position, row and
// store after each other (of a write's row only the place depends on the position: it could be asked for at once).
struct RowsSpot {
    int s, t, slot;  // slot -1: nothing there (a write: no row; a read: zeros), t -1: no row
};
template <bool READ>
__device__ __forceinline__ RowsSpot rows_spot(const KvRowsArgs& a, int m) {
    const int ring = a.c.cap - a.c.sinks, s = a.T == 1 ? m : m / a.T, t = m - s * a.T;
    const SeqSpan q = seq_span(a.pos, a.counts, s, a.T);
    const int p = q.pos + t, end = READ && a.lens ? min(max(a.lens[s], 0), kKvMaxPos) : q.end;
    // of two tokens of a call that share a slot the later one is written
    const bool held = p >= 0 && p < end && (p < a.c.sinks || p >= end - ring);
    return {s, t < q.count ? t : -1, held ? kv_slot(p, a.c.sinks, ring) : -1};
}

template <int DH, class T, int U>
__global__ __launch_bounds__(256) void kv_write_kernel(KvRowsArgs a) {
    constexpr int LR = DH / 8, rows = 256 / LR;
    const int tokens = a.c.n * a.T, h0 = blockIdx.y * U, row_in = threadIdx.x / LR, l = threadIdx.x % LR;
    if (256 % LR && row_in >= rows) return;
    const KvRows& x = blockIdx.z ? a.v : a.k;
    uint8_t* codes = blockIdx.z ? a.c.v : a.c.k;
    uint8_t* scales = blockIdx.z ? a.c.vs : a.c.ks;
    for (long long m = (long long)blockIdx.x * rows + row_in; m < tokens; m += (long long)gridDim.x * rows) {
        const RowsSpot r = rows_spot<false>(a, (int)m);
        if (r.t < 0 || r.slot < 0) continue;  // (the four lanes of a block together)
        const T* from = (const T*)x.data + r.s * x.seq + r.t * x.token + 8 * l;
        const size_t to = ((size_t)r.s * a.c.heads + h0) * a.c.cap + r.slot;
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (h0 + u < a.c.heads) real_load8<T>(from + (h0 + u) * x.head, 8, v[u]);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (h0 + u >= a.c.heads) break;
            uint32_t sb;
            const uint32_t w = mx4_block(v[u], sb);
            const size_t row = to + (size_t)u * a.c.cap;
            *(uint32_t*)(codes + row * (DH / 2) + 4 * l) = w;
            if ((l & 3) == 0) scales[row * (DH / 32) + (l >> 2)] = (uint8_t)sb;
        }
    }
}

template <int DH, class T, int U>
__global__ __launch_bounds__(256) void kv_read_kernel(KvRowsArgs a) {
    constexpr int LR = DH / 8, rows = 256 / LR;
    const int tokens = a.c.n * a.T, h0 = blockIdx.y * U, row_in = threadIdx.x / LR, l = threadIdx.x % LR;
    if (256 % LR && row_in >= rows) return;
    const KvRows& x = blockIdx.z ? a.v : a.k;
    const uint8_t* codes = blockIdx.z ? a.c.v : a.c.k;
    const uint8_t* scales = blockIdx.z ? a.c.vs : a.c.ks;
    for (long long m = (long long)blockIdx.x * rows + row_in; m < tokens; m += (long long)gridDim.x * rows) {
        const RowsSpot r = rows_spot<true>(a, (int)m);
        if (r.t < 0) continue;
        T* to = (T*)x.data + r.s * x.seq + r.t * x.token + 8 * l;
        const size_t from = ((size_t)r.s * a.c.heads + h0) * a.c.cap + max(r.slot, 0);
        uint32_t w[U], sb[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            w[u] = sb[u] = 0;
            if (h0 + u >= a.c.heads || r.slot < 0) continue;
            const size_t row = from + (size_t)u * a.c.cap;
            w[u] = *(const uint32_t*)(codes + row * (DH / 2) + 4 * l);
            sb[u] = scales[row * (DH / 32) + (l >> 2)];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (h0 + u >= a.c.heads) break;
            float v[8];
            mx4_unpack8(w[u], mx4_scale(sb[u]), v);
            real_store8<T>(to + (h0 + u) * x.head, 8, v);
        }
    }
}

template <class F>
auto by_width(int dh, F&& f) {
    switch (dh) {
        case 32: return f(std::integral_constant<int, 32>());
        case 64: return f(std::integral_constant<int, 64>());
        case 96: return f(std::integral_constant<int, 96>());
        default: return f(std::integral_constant<int, 128>());
    }
}

template <bool READ>
hipError_t launch_rows(const KvRowsArgs& a, hipStream_t s) {
    const int rows = 256 / (a.c.dh / 8);
    const long long groups = ((long long)a.c.n * a.T + rows - 1) / rows;
    // four heads a lane where that leaves four workgroups a CU
    const bool many = groups * a.c.heads >= 2048;
    const dim3 grid((unsigned)std::min<long long>(groups, 1 << 16), many ? (a.c.heads + 3) / 4 : a.c.heads, 2);
    return by_width(a.c.dh, [&](auto w) {
        constexpr int DH = decltype(w)::value;
        return by_real(a.type, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            const auto go = [&](auto u) {
                constexpr int U = decltype(u)::value;
                if constexpr (READ) hipLaunchKernelGGL((kv_read_kernel<DH, T, U>), grid, dim3(256), 0, s, a);
                else hipLaunchKernelGGL((kv_write_kernel<DH, T, U>), grid, dim3(256), 0, s, a);
                return hipGetLastError();
            };
            return many ? go(std::integral_constant<int, 4>()) : go(std::integral_constant<int, 1>());
        });
    });
}

// ---- attention -----------------------------------------------------------------------------------------------------
// The cache is read in tiles of 32 slots. The tiles that hold a position some row of a row tile sees, in slot order: up to
// three runs (the sinks; the ring's part up to the newest position; the older part behind it, where the run wraps).
struct Tiles {
    int n0, n1, n2;      // tiles of each run
    int b1, b2;          // first tiles of the second and third
    __device__ __forceinline__ int count() const { return n0 + n1 + n2; }
    __device__ __forceinline__ int at(int o) const { return o + (o >= n0 ? b1 - n0 : 0) + (o >= n0 + n1 ? b2 - b1 - n1 : 0); }
};
template <class T>
struct Terms;  // bf16 parts that hold a query element, and those that a probability is split into
template <>
struct Terms<float> { static constexpr int q = 3, p = 3; };
template <>
struct Terms<_Float16> { static constexpr int q = 2, p = 2; };
template <>
struct Terms<__bf16> { static constexpr int q = 1, p = 2; };

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const mx_v2bf v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Eight floats as N bf16 vectors whose sum is them (to 8 N bits).
template <int N>
__device__ __forceinline__ void split_bf16(const float x[8], v8bf out[N]) {
    uint32_t w[N][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int n = 0; n < N; n++) {
            w[n][i] = pack_bf16(a, b);
            if (n + 1 < N) {
                a -= bf16_lo(w[n][i]);
                b -= bf16_hi(w[n][i]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < N; n++) out[n] = __builtin_bit_cast(v8bf, *(uint4*)w[n]);
}

// Channels of a head as the two products take them, with i = lane & 15 and g = lane >> 4.
//   Scores, K (16 slots a product) times q: step s of DH / 32 covers, for lane group g, channels (DH / 4) g + 8 s .. + 7, so
//   that a lane's steps are neighbouring words of a row (DH 96: channels 32 s + 8 g, since 24 do not end with a block).
//   Output, V^T times the probabilities: channels in chunks of 16 E, lane i owning E neighbouring ones (E 8, 4, 2), a pair at a
//   time.
template <int DH>
struct Width {
    static constexpr int KS = DH / 32, NB = DH / 32, NA = DH / 32;  // NA: fragments of the output, 16 pairs of channels each
    static constexpr bool kEven = DH != 96;
    static constexpr int KW = kEven ? 1 : 3;  // scale bytes a lane needs of a key
    static constexpr int chunks = DH == 96 ? 2 : 1;
    static constexpr int E0 = DH == 96 ? 4 : DH / 16;
    __host__ __device__ static constexpr int E(int c) { return c == 0 ? E0 : 2; }
    __host__ __device__ static constexpr int base(int c) { return c == 0 ? 0 : 64; }
    __host__ __device__ static constexpr int a0(int c) { return c == 0 ? 0 : E0 / 2; }
    __device__ static int k_channel(int g, int s) { return kEven ? (DH / 4) * g + 8 * s : 32 * s + 8 * g; }
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A scale of the byte at bit 8 b of a word, for a conversion: it reads the exponent bits alone, so the byte is only rotated there.
__device__ __forceinline__ float scale_at(uint32_t w, int shift) { return __uint_as_float(__builtin_amdgcn_alignbit(w, w, shift)); }
__device__ __forceinline__ constexpr int scale_shift(int b) { return (8 * b + 9) & 31; }

// Of two lanes 16 (32) apart, both their values.
__device__ __forceinline__ float max_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

constexpr int kTile = 32;
constexpr float kLog2e = 1.4426950408889634f;

// One 16-byte (4-byte) load per lane from global memory straight into LDS: lane L's bytes land at LDS offset lds + AT + 16 L
// (lds + 4 L). Inline assembly, with the waits written out (vm_wait), because the compiler would wait for all such loads before
// any LDS read. The LDS address goes through M0; the s_nop covers the wait states after a vector instruction's write of the
// scalar base and after that of M0. AT counts on both sides. No register receives anything. (nt: a tile is read once; 12 % more
// bandwidth than without for plain reads of large arrays.)
template <int AT>
__device__ __forceinline__ void lds_load16(const uint8_t* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1 offset:%3 nt" ::"v"(off), "s"(base), "s"(lds), "i"(AT) : "m0", "memory");
}
__device__ __forceinline__ void lds_load16(const uint8_t* p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(p), "s"(lds) : "m0", "memory");
}
__device__ __forceinline__ void lds_load4(const uint8_t* p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 3\n\tglobal_load_lds_dword %0, off nt" ::"v"(p), "s"(lds) : "m0", "memory");
}
template <int N>
__device__ __forceinline__ void vm_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

// A tile of 32 slots of one head in LDS: K's rows, V's rows, their scales, in DH / 32 loads of 1 KiB and one of 256 bytes (which
// the scales of narrower heads do not fill). The order is chosen against bank conflicts: of K, block b of slot j stands at
// place b ^ f(j) of its row (DH 128; f from bits 1 and 3 of j, in which the eight slots that eight lanes read together differ
// besides bit 0), of V slot j's row is row j ^ ((j >> 3) & 3) (the four lane groups read slots eight apart).
template <int DH>
struct KvTile {
    using W = Width<DH>;
    static constexpr int row = DH / 2, half = 32 * row, o_scales = 2 * half, bytes = o_scales + 256;
    static constexpr int loads = W::KS + 1;

    __device__ static __forceinline__ int k_place(int j) { return DH == 128 ? ((j >> 1) & 1) | ((j >> 2) & 2) : 0; }

    // What each lane loads of a tile, from the tile's place in the planes. Where a load is of K or V alone (DH 64 and 128) the place
    // is a scalar; otherwise it is added to each lane's address.
    struct Source {
        uint32_t k_off, v_off;         // within 1 KiB of K and V
        const uint8_t* codes[W::KS];   // DH 32 and 96
        const uint8_t* scales;
        __device__ __forceinline__ void set(const KvCache& c, int lane) {
            if constexpr (DH % 64 == 0) {
                const int j = 16 * lane / row, b = 16 * lane % row;
                k_off = j * row + (b ^ (16 * k_place(j)));
                v_off = (j ^ ((j >> 3) & 3)) * row + b;
            } else {
#pragma unroll
                for (int x = 0; x < W::KS; x++) {
                    const int at = 1024 * x + 16 * lane, in = at < half ? at : at - half, j = in / row;
                    codes[x] = at < half ? c.k + in : c.v + (j ^ ((j >> 3) & 3)) * row + in % row;
                }
            }
            const int at = min(4 * (W::NB == 3 ? lane : lane & (16 * W::NB - 1)), 64 * W::NB - 4);  // (lanes past the scales repeat some)
            scales = at < 32 * W::NB ? c.ks + at : c.vs + at - 32 * W::NB;
        }
        __device__ __forceinline__ void load(const KvCache& c, size_t slot, uint32_t lds) const {
            if constexpr (DH % 64 == 0) {
                const uint8_t *k = c.k + slot * row, *v = c.v + slot * row;
                lds_load16<0>(k, k_off, lds);
                if constexpr (DH == 128) lds_load16<1024>(k, k_off, lds);
                lds_load16<0>(v, v_off, lds + half);
                if constexpr (DH == 128) {
                    // (slots 16 and on: the same order, since bits 3 and 4 of a slot choose the row)
                    lds_load16<1024>(v, v_off ^ (2 * row), lds + half);
                }
            } else {
#pragma unroll
                for (int x = 0; x < W::KS; x++) lds_load16(codes[x] + slot * row, lds + 1024 * x);
            }
            lds_load4(scales + slot * W::NB, lds + o_scales);
        }
    };

    // Product h of the scores: lane i holds slot 8 (i >> 2) + 4 h + (i & 3), so that the scores of slots 8 g .. 8 g + 7 come out in
    // lane group g.
    struct Key {
        uint32_t w[W::KS], s[W::KW];
        __device__ __forceinline__ void read(const uint8_t* p, int h, int i, int g) {
            const int j = (i >> 2) * 8 + 4 * h + (i & 3);
            const uint8_t* q = p + j * row;
            if constexpr (DH == 128) *(u32x4*)w = *(const u32x4*)(q + 16 * (g ^ k_place(j)));
            else if constexpr (DH == 64) *(u32x2*)w = *(const u32x2*)(q + 8 * g);
            else
#pragma unroll
                for (int x = 0; x < W::KS; x++) w[x] = *(const uint32_t*)(q + 16 * x + 4 * g);
#pragma unroll
            for (int x = 0; x < W::KW; x++) s[x] = p[o_scales + j * W::NB + (W::kEven ? (DH / 4) * g / 32 : x)];
        }
    };
    // Slots 8 g .. 8 g + 7, the lane's channels of each.
    struct Value {
        uint32_t w[W::chunks][8];
        uint32_t s[2 * W::NB];
        __device__ __forceinline__ void read(const uint8_t* p, int i, int g) {
#pragma unroll
            for (int c = 0; c < W::chunks; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint8_t* q = p + half + (8 * g + (e ^ g)) * row + (W::base(c) + i * W::E(c)) / 2;
                    w[c][e] = W::E(c) == 8 ? *(const uint32_t*)q : W::E(c) == 4 ? *(const uint16_t*)q : *q;
                }
#pragma unroll
            for (int x = 0; x < W::NB; x++) *(u32x2*)(s + 2 * x) = *(const u32x2*)(p + o_scales + 32 * W::NB + 8 * g * W::NB + 8 * x);
        }
        // Slot 8 g + e as zeros.
        __device__ __forceinline__ void drop(int e) {
#pragma unroll
            for (int c = 0; c < W::chunks; c++) w[c][e] = 0;
#pragma unroll
            for (int b = 0; b < W::NB; b++) {
                const int at = e * W::NB + b;
                s[at >> 2] &= ~(255u << (8 * (at & 3)));
            }
        }
        // The scale byte of slot 8 g + e for block b, and the scale for a conversion (of this lane's channels in chunk c).
        __device__ __forceinline__ uint32_t byte(int e, int b) const {
            const int at = e * W::NB + b;
            return (s[at >> 2] >> (8 * (at & 3))) & 255;
        }
        __device__ __forceinline__ float scale(int c, int e, int i) const {
            if constexpr (DH == 128) return scale_at(s[e], 8 * (i >> 2) + 9);
            else if constexpr (DH == 64) return scale_at(s[e >> 1], 16 * (e & 1) + 8 * (i >> 3) + 9);
            else if constexpr (DH == 32) return scale_at(s[e >> 2], scale_shift(e & 3));
            else {
                if (c == 1) return scale_at(s[(3 * e + 2) >> 2], scale_shift((3 * e + 2) & 3));
                const int at = 3 * e;  // this byte or the next
                const float lo = scale_at(s[at >> 2], scale_shift(at & 3)), hi = scale_at(s[(at + 1) >> 2], scale_shift((at + 1) & 3));
                return i & 8 ? hi : lo;
            }
        }
    };
};

// Two elements of word w (byte b), scaled, as bf16.
__device__ __forceinline__ uint32_t unpack2(uint32_t w, float s, int b) {
    switch (b) {
        case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
        case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
        case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
        default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
    }
}

// What a wave's rows and the slots are, for the masks. Uniform but for `at` and `low`.
struct Seen {
    int sinks, ring, window;
    int last, newest;     // the last position, and its slot in the ring (-1: none is there)
    int lo_at, hi_at;     // positions of the wave's rows
    int at;               // of this lane's row
    int low;              // the last position behind its window
    // The position that a slot holds, if that is one of a sink or from `sinks` on.
    __device__ __forceinline__ int position(int j) const {
        const int back = newest - j;
        return j < sinks ? j : last - (back + (back < 0 ? ring : 0));
    }
    __device__ __forceinline__ bool holds(int j) const {
        const int p = position(j);
        return (p >= (j < sinks ? 0 : sinks)) & (p <= last);
    }
    // A row at position at, which sees no position up to low but the sinks'.
    __device__ __forceinline__ bool sees(int j, int at, int low) const {
        const int p = position(j);
        return (p >= (j < sinks ? 0 : sinks)) & (p <= at) & (p <= last) & ((j < sinks) | (p > low));
    }
    // Of a tile: its slots hold 32 positions in a row, from which on (-1: not so).
    __device__ __forceinline__ int run(int j0) const {
        if (j0 < sinks || (j0 <= newest && newest < j0 + 31)) return -1;
        const int p = position(j0);
        return p >= sinks && p + 31 <= last ? p : -1;
    }
    // Every row sees every slot of the tile.
    __device__ __forceinline__ bool whole(int j0) const {
        if (j0 + 31 < sinks) return j0 + 31 <= lo_at;
        const int p = run(j0);
        return p >= 0 && p + 31 <= lo_at && (window <= 0 || p > hi_at - window);
    }
};

__device__ __forceinline__ Tiles tiles_of(const Seen& q, int cap) {
    Tiles r{0, 0, 0, 0, 0};
    if (q.hi_at < 0) return r;
    r.n0 = (min(q.sinks, q.hi_at + 1) + 31) >> 5;
    int lo = max(q.sinks, q.last + 1 - q.ring);
    if (q.window > 0) lo = max(lo, q.lo_at - q.window + 1);
    if (q.hi_at < lo) return r;
    // (both are within a ring of the last position: no division)
    const auto slot = [&](int p) {
        const int j = q.newest - (q.last - p);
        return j < q.sinks ? j + q.ring : j;
    };
    const int first = slot(lo), newest = slot(q.hi_at);
    const int a = first >> 5, b = (newest >> 5) + 1;
    const bool wraps = first > newest;
    r.b1 = max(r.n0, wraps ? q.sinks >> 5 : a);
    r.n1 = max(0, b - r.b1);
    if (wraps) {
        r.b2 = max(max(r.n0, r.b1 + r.n1), a);
        r.n2 = max(0, (cap >> 5) - r.b2);
    }
    return r;
}

// Running softmax of 8 rows, a lane's share: column i = lane & 15 of the products is row i >> 1; O^T in the second product's layout for
// each of HB heads (a column's own head counts); the maximum of the row (common to the lanes that have it), and the sum over
// the lane's own slots.
template <int DH, int HB>
struct RowState {
    v4f acc[HB][Width<DH>::NA];
    float m, l;
    uint32_t nan_blocks;  // careful form: bit b: a key that the row sees has NaN in channels 32 b .. 32 b + 31
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int hb = 0; hb < HB; hb++)
#pragma unroll
            for (int d = 0; d < Width<DH>::NA; d++) acc[hb][d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        m = -INFINITY;
        l = 0.0f;
        nan_blocks = 0;
    }
};

// One tile of HB heads for 8 rows, column i of the products belonging to head `mine` of them.
//
// Scores: product h of a head leaves lane (i, g) with row i >> 1 and slots 8 g + 4 h .. + 3 of the tile. With several heads each
// product is formed for all columns and kept for its own, so that the softmax between is done once for all of them.
//
// Output: unpacking a byte of V gives two neighbouring channels of one slot in a register, where the product wants two
// neighbouring entries of the sum. They are taken as such: the sum runs over (slot, channel parity), and the column of even
// parity has the probability at the slot's even entry and zero at its odd one, the other column the reverse. A row thus has two
// columns, which give its even and its odd channels; no value is moved between lanes or registers on the way, and the
// probabilities stay in the lane where the scores came out.
//
// CAREFUL keeps blocks of NaN out of the product (they would spread over rows that do not see their key) and notes who sees them
// instead.
template <int DH, class T, int HB, bool CAREFUL>
__device__ __forceinline__ void tile_step(RowState<DH, HB>& st, const uint8_t* tile, const v8bf (*qf)[Terms<T>::q], float scale,
                                          const Seen& seen, int j0, bool whole, int i, int g, int mine) {
    using W = Width<DH>;
    using Tile = KvTile<DH>;
    constexpr int QT = Terms<T>::q, PT = Terms<T>::p;
    float sc[8];
#pragma unroll
    for (int hb = 0; hb < HB; hb++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            typename Tile::Key x;
            x.read(tile + hb * Tile::bytes, h, i, g);
            v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < W::KS; s++) {
                const float ks = mx4_scale(x.s[W::kEven ? 0 : s]);
                uint32_t kw[4];
#pragma unroll
                for (int b = 0; b < 4; b++) kw[b] = unpack2(x.w[s], ks, b);
                const v8bf kf = __builtin_bit_cast(v8bf, *(u32x4*)kw);
#pragma unroll
                for (int n = QT - 1; n >= 0; n--) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[s][n], d, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) sc[4 * h + r] = hb == 0 || mine == hb ? d[r] : sc[4 * h + r];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) sc[e] *= scale;
    uint32_t sees = 255, drop = 0;
    if (!whole) {
        asm volatile("");  // a branch: as selects this would cost every tile
        sees = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int j = j0 + 8 * g + e;
            const bool held = seen.holds(j), v = seen.sees(j, seen.at, seen.low);
            sees |= (uint32_t)v << e;
            drop |= (uint32_t)!held << e;  // never written, or lost: may hold anything
            sc[e] = v ? sc[e] : -INFINITY;
        }
    }
    const float mt = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
    if (__any(mt > st.m)) {  // rare after the first tiles
        const float mn = fmaxf(st.m, max_groups(mt)), al = __builtin_amdgcn_exp2f(mn == -INFINITY ? 0.0f : st.m - mn);
        st.m = mn;
        st.l *= al;
#pragma unroll
        for (int hb = 0; hb < HB; hb++)
#pragma unroll
            for (int d = 0; d < W::NA; d++) st.acc[hb][d] *= al;
    }
    const float mu = st.m == -INFINITY ? 0.0f : st.m;
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(sc[e] - mu);
    st.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    // the probabilities in PT parts, each at its parity's half of a word
    const uint32_t parity = i & 1 ? 0xffff0000u : 0x0000ffffu;
    uint32_t pw[PT][8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float x = p[e];
#pragma unroll
        for (int n = 0; n < PT; n++) {
            const uint32_t both = pack_bf16(x, x);
            pw[n][e] = both & parity;
            if (n + 1 < PT) x -= bf16_hi(both);
        }
    }
#pragma unroll
    for (int hb = 0; hb < HB; hb++) {
        typename Tile::Value x;
        x.read(tile + hb * Tile::bytes, i, g);
        if (!whole) {
            asm volatile("");
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (drop >> e & 1) x.drop(e);
        }
        if (CAREFUL) {
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int b = 0; b < W::NB; b++)
                    if (((sees >> e) & 1) && mine == hb && x.byte(e, b) > 252u) st.nan_blocks |= 1u << b;
        }
#pragma unroll
        for (int c = 0; c < W::chunks; c++) {
            float vs[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                vs[e] = x.scale(c, e, i);
                // (the writer's scales are at most 252, or 255 for NaN)
                if (CAREFUL && (__float_as_uint(vs[e]) >> 23 & 255) > 252u) {
                    x.w[c][e] = 0;
                    vs[e] = 0.0f;
                }
            }
#pragma unroll
            for (int b = 0; b < W::E(c) / 2; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t vw[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) vw[r] = unpack2(x.w[c][4 * h + r], vs[4 * h + r], b);
                    const v8bf vf = __builtin_bit_cast(v8bf, *(u32x4*)vw);
                    v4f& o = st.acc[hb][W::a0(c) + b];
#pragma unroll
                    for (int n = PT - 1; n >= 0; n--)
                        o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(v8bf, *(u32x4*)(pw[n] + 4 * h)), o, 0, 0, 0);
                }
        }
    }
}

// Parts of a row for the join: sums, then maximum and sum of probabilities.
template <int DH>
constexpr int kPart = DH + 4;

// Rows of a wave: half the columns of a product.
constexpr int kRows = 8;

// Stages of a wave's tiles in LDS, for two workgroups of four waves a CU.
template <int DH, int HB>
struct Stages {
    static constexpr int bytes = HB * KvTile<DH>::bytes;
    static constexpr int n = std::min(4, std::max(2, 20 * 1024 / bytes));
    static constexpr int loads = HB * KvTile<DH>::loads;
    static constexpr int wave = n * bytes;
    static_assert((n - 1) * loads <= 63, "");
};

// Few query rows: a wave takes up to 8 rows of one sequence over a share of the tiles: a row tile of one key/value head (its
// query heads, token after token), or, with HB > 1, all rows of HB heads (8 or fewer). Tiles come straight into the wave's own
// LDS stages, up to three ahead. WAVES waves share the tiles (of one chunk of them, where there are several) and add up what
// they have in LDS; with WAVES 1 a wave is alone with its rows.
//
// Bound by reading the cache, with the unpacking close behind. 32 conversations of 16384 positions (8 heads of 128, four query
// heads each, bf16): 101 us, 5.6 TB/s; of 1 to 16384 positions, 276 MB, 71 us (3.9 TB/s: the lengths do not divide evenly over the
// chip) and 4.5 for the join; 256 windows of 1000 (8 heads of 64, two query heads each, fp16, 109 MB) 29 us; 4096 windows of 64 (8
// fp32 heads of 32, 57 MB) 24 us, where a wave's life is mostly its first tiles' latency; one conversation of 30000 (33 MB) 13 us and
// 6 for the join: two heads a wave make 236 workgroups of it, where 512 have room, each with sixteen tiles one after another.
template <int DH, class T, int HB, int WAVES>
__global__ __launch_bounds__(256, 2) void kv_attention_rows_kernel(KvAttnArgs a, int row_tiles, int chunk_tiles) {
    using W = Width<DH>;
    using Tile = KvTile<DH>;
    using St = Stages<DH, HB>;
    constexpr int QT = Terms<T>::q, LD = DH + 4;
    static_assert(4 * kRows * (LD + 2) * 4 <= 4 * St::wave, "");
    __shared__ __align__(16) uint8_t smem[4 * St::wave];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = WAVES > 1 ? blockIdx.x : blockIdx.x * 4 + wave, w = WAVES > 1 ? wave : 0;
    const int blocks = a.c.heads / HB, units = a.c.n * blocks * row_tiles;
    if (unit >= units) return;
    const int pair = row_tiles == 1 ? unit : unit / row_tiles, rt = unit - pair * row_tiles;
    const int s = blocks == 1 ? pair : pair / blocks, h0 = (pair - s * blocks) * HB;
    const SeqSpan q = seq_span(a.pos, a.counts, s, a.T);
    const int ring = a.c.cap - a.c.sinks, sinks = a.c.sinks;
    const int t_lo = rt == 0 ? 0 : rt * kRows / a.group;
    if (t_lo >= q.count) return;
    const int t_hi = a.T == 1 ? 0 : min((rt * kRows + kRows - 1) / a.group, q.count - 1);

    Seen seen;
    seen.sinks = sinks; seen.ring = ring; seen.window = a.window;
    seen.last = q.end - 1;
    seen.newest = seen.last >= sinks ? kv_slot(seen.last, sinks, ring) : -1;
    seen.lo_at = q.pos + t_lo;
    seen.hi_at = q.pos + t_hi;
    const Tiles tl = tiles_of(seen, a.c.cap);
    const int n_tiles = tl.count();
    const int o0 = blockIdx.y * chunk_tiles, o1 = min(n_tiles, o0 + chunk_tiles);
    if (blockIdx.y && o0 >= n_tiles) return;

    typename Tile::Source src;
    src.set(a.c, lane);
    uint8_t* own = smem + wave * St::wave;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)own;
    const size_t plane = (size_t)(s * a.c.heads + h0) * a.c.cap;
    auto load = [&](int o, int stage) {
        const size_t slot = plane + tl.at(o) * kTile;
#pragma unroll
        for (int hb = 0; hb < HB; hb++) src.load(a.c, slot + (size_t)hb * a.c.cap, lds0 + stage * St::bytes + hb * Tile::bytes);
    };
    // the first tiles of a pass are on their way
    auto start = [&] {
#pragma unroll
        for (int x = 0; x < St::n - 1; x++)
            if (o0 + w + x * WAVES < o1) load(o0 + w + x * WAVES, x);
    };
    start();

    // this lane's row
    const int rows = a.T * a.group;  // of a head
    const int col = i >> 1, hb_own = HB > 1 ? col / rows : 0, row = HB > 1 ? col - hb_own * rows : rt * kRows + col;
    const int t = a.T == 1 ? 0 : row / a.group, head = (h0 + hb_own) * a.group + (row - t * a.group);
    const bool there = hb_own < HB && row < rows && t < q.count;
    seen.at = q.pos + t;
    seen.low = a.window > 0 ? seen.at - a.window : INT_MIN;
    v8bf qf[W::KS][QT];
#pragma unroll
    for (int st = 0; st < W::KS; st++) {
        float x[8] = {};
        if (there) real_load8<T>((const T*)a.q.data + s * a.q.seq + t * a.q.token + head * a.q.head + W::k_channel(g, st), 8, x);
        split_bf16<QT>(x, qf[st]);
    }
    const float scale = a.scale * kLog2e;

    RowState<DH, HB> st;
    auto sweep = [&](auto careful) {
        st.clear();
        int stage = 0;
        for (int o = o0 + w; o < o1; o += WAVES) {
            // the tiles issued after this one: up to n - 2 now, one more below
            const int more = (o1 - 1 - o) / WAVES;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last stage's reads are done: it is loaded anew
            if (more >= St::n - 1) {
                load(o + (St::n - 1) * WAVES, stage == 0 ? St::n - 1 : stage - 1);
                vm_wait<(St::n - 1) * St::loads>();
            } else if (St::n > 3 && more == 2) {
                vm_wait<2 * St::loads>();
            } else if (St::n > 2 && more == 1) {
                vm_wait<St::loads>();
            } else {
                vm_wait<0>();
            }
            const int j0 = __builtin_amdgcn_readfirstlane(tl.at(o) * kTile);
            tile_step<DH, T, HB, decltype(careful)::value>(st, own + stage * St::bytes, qf, scale, seen, j0, seen.whole(j0), i, g, hb_own);
            stage = stage == St::n - 1 ? 0 : stage + 1;
        }
    };
    // the lane's sums: of its row's own head
    v4f acc[W::NA];
    auto pick = [&] {
#pragma unroll
        for (int d = 0; d < W::NA; d++) {
            acc[d] = st.acc[0][d];
#pragma unroll
            for (int hb = 1; hb < HB; hb++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[d][r] = hb_own == hb ? st.acc[hb][d][r] : acc[d][r];
        }
    };
    sweep(std::false_type());
    pick();
    {
        // A NaN among the sums: it may come from a value that the row does not see.
        float bad = 0.0f;
#pragma unroll
        for (int d = 0; d < W::NA; d++)
#pragma unroll
            for (int r = 0; r < 4; r++) bad += acc[d][r] * 0.0f;
        if (__any(bad != 0.0f)) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            start();
            sweep(std::true_type());
            pick();
            st.nan_blocks |= __shfl_xor(st.nan_blocks, 16, 64);
            st.nan_blocks |= __shfl_xor(st.nan_blocks, 32, 64);
#pragma unroll
            for (int c = 0; c < W::chunks; c++)
#pragma unroll
                for (int b = 0; b < W::E(c) / 2; b++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if ((st.nan_blocks >> ((W::base(c) + (4 * g + r) * W::E(c)) / 32)) & 1) acc[W::a0(c) + b][r] = NAN;
        }
    }
    st.l = sum_groups(st.l);
    const bool split = n_tiles > chunk_tiles;
    // [chunk][unit][column][kPart]
    float* part = a.ws + (((size_t)blockIdx.y * units + unit) * kRows) * kPart<DH>;
    if constexpr (WAVES == 1) {
        const float f = st.l == 0.0f ? 0.0f : 1.0f / st.l;
        T* out = (T*)a.out.data + s * a.out.seq + t * a.out.token + head * a.out.head;
        // Lanes 2 r and 2 r + 1 have the even and odd channels of element groups 0 .. 3: the first gets both of groups 0 and 1, the
        // second those of groups 2 and 3.
        const bool odd = i & 1;
#pragma unroll
        for (int c = 0; c < W::chunks; c++) {
            float v[2][W::E0];
#pragma unroll
            for (int b = 0; b < W::E(c) / 2; b++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const v4f& x = acc[W::a0(c) + b];
                    const float keep = odd ? x[2 + r] : x[r], get = dpp_move<0xB1>(odd ? x[r] : x[2 + r]);
                    v[r][2 * b] = (odd ? get : keep) * f;
                    v[r][2 * b + 1] = (odd ? keep : get) * f;
                }
            if (there) {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    T* p = out + W::base(c) + (4 * g + 2 * (i & 1) + r) * W::E(c);
                    const float* from = v[r];
                    if (W::E(c) == 8) {
                        real_store8<T>(p, 8, from);
                    } else if (W::E(c) == 4) {
                        real_store4(p, from, 4);
                    } else {
                        const T u[2] = {(T)from[0], (T)from[1]};
                        __builtin_memcpy(p, u, sizeof(u));
                    }
                }
            }
        }
    } else {
        // join the waves: their sums at the largest maximum, added in the waves' order (the stages are done with)
        float* s_o = (float*)smem;                                    // [wave][column][LD]
        float (*s_ml)[2][kRows] = (float (*)[2][kRows])(s_o + WAVES * kRows * LD);
        __syncthreads();
        if (g == 0 && (i & 1) == 0) {
            s_ml[w][0][col] = st.m;
            s_ml[w][1][col] = st.l;
        }
        __syncthreads();
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < WAVES; x++) top = fmaxf(top, s_ml[x][0][col]);
        const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - top);
#pragma unroll
        for (int c = 0; c < W::chunks; c++)
#pragma unroll
            for (int b = 0; b < W::E(c) / 2; b++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    s_o[(w * kRows + col) * LD + W::base(c) + (4 * g + r) * W::E(c) + 2 * b + (i & 1)] = acc[W::a0(c) + b][r] * f;
        __syncthreads();
        const int keep = min(kRows, HB > 1 ? HB * rows : rows - rt * kRows);
        for (int x = threadIdx.x * 4; x < keep * DH; x += 256 * 4) {
            const int cc = x / DH, d = x - cc * DH;
            const int hh = HB > 1 ? cc / rows : 0, rr = HB > 1 ? cc - hh * rows : rt * kRows + cc;
            const int tt = a.T == 1 ? 0 : rr / a.group, hd = (h0 + hh) * a.group + (rr - tt * a.group);
            if (tt >= q.count) continue;
            float most = -INFINITY, total = 0.0f;
#pragma unroll
            for (int y = 0; y < WAVES; y++) most = fmaxf(most, s_ml[y][0][cc]);
            v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int y = 0; y < WAVES; y++) {
                total += s_ml[y][1][cc] * (most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_ml[y][0][cc] - most));
                sum += *(const v4f*)(s_o + (y * kRows + cc) * LD + d);
            }
            if (split) {
                *(v4f*)(part + cc * kPart<DH> + d) = sum;
                if (d == 0) {
                    part[cc * kPart<DH> + DH] = most;
                    part[cc * kPart<DH> + DH + 1] = total;
                }
            } else {
                real_store4((T*)a.out.data + s * a.out.seq + tt * a.out.token + hd * a.out.head + d, sum * (total == 0.0f ? 0.0f : 1.0f / total), 4);
            }
        }
    }
}

// Joins the chunks of a row that took more than one: a wave a row, its lanes over channels (four each) and, in as many groups as fit,
// over the chunks, whose sums are added in a fixed order. Units have `per` rows. (4.5 us for 32 conversations of 32 query heads, 6 for
// the 59 chunks of one long one: its latency.)
template <int DH, class T>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(KvAttnArgs a, int per, int hb, int row_tiles, int chunk_tiles) {
    constexpr int LC = DH / 4, G = 64 / LC;  // lanes a group, groups
    const int lane = threadIdx.x & 63, col = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = blockIdx.x;
    const int blocks = a.c.heads / hb, units = a.c.n * blocks * row_tiles;
    const int pair = row_tiles == 1 ? unit : unit / row_tiles, rt = unit - pair * row_tiles;
    const int s = pair / blocks, h0 = (pair - s * blocks) * hb;
    const SeqSpan q = seq_span(a.pos, a.counts, s, a.T);
    const int rows = a.T * a.group;
    if (col >= (hb > 1 ? hb * rows : per)) return;
    const int hh = hb > 1 ? col / rows : 0, row = hb > 1 ? col - hh * rows : rt * per + col;
    const int t = row / a.group, head = (h0 + hh) * a.group + (row - t * a.group);
    if (row >= rows || t >= q.count) return;
    Seen seen;
    seen.sinks = a.c.sinks; seen.ring = a.c.cap - a.c.sinks; seen.window = a.window;
    seen.last = q.end - 1;
    seen.newest = seen.last >= seen.sinks ? kv_slot(seen.last, seen.sinks, seen.ring) : -1;
    seen.lo_at = q.pos + rt * per / a.group;
    seen.hi_at = q.pos + min((rt * per + per - 1) / a.group, q.count - 1);
    const int chunks = (tiles_of(seen, a.c.cap).count() + chunk_tiles - 1) / chunk_tiles;
    if (chunks <= 1) return;
    const size_t step = (size_t)units * per * kPart<DH>;
    const float* part = a.ws + ((size_t)unit * per + col) * kPart<DH>;
    float top = -INFINITY;
    for (int c = lane; c < chunks; c += 64) top = fmaxf(top, part[c * step + DH]);
    top = wave_max(top);
    const float tu = top == -INFINITY ? 0.0f : top;
    const int grp = lane / LC, d = (lane - grp * LC) * 4;
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float total = 0.0f;
#pragma unroll 4
    for (int c = grp < G ? grp : chunks; c < chunks; c += G) {
        const float f = __builtin_amdgcn_exp2f(part[c * step + DH] - tu);
        sum += *(const v4f*)(part + c * step + d) * f;
        total += part[c * step + DH + 1] * f;
    }
    v4f all = sum;
    float norm = total;
#pragma unroll
    for (int x = 1; x < G; x++) {
#pragma unroll
        for (int r = 0; r < 4; r++) all[r] += __shfl(sum[r], lane + x * LC, 64);
        norm += __shfl(total, lane + x * LC, 64);
    }
    if (lane < LC)
        real_store4((T*)a.out.data + s * a.out.seq + t * a.out.token + head * a.out.head + d, all * (norm == 0.0f ? 0.0f : 1.0f / norm), 4);
}

// ---- many query rows ----
// A workgroup of four waves takes 128 query rows of one key/value head (the heads of its group, token after token), a wave 32 of
// them. Tiles of 32 slots come into LDS as they are, three ahead; the workgroup unpacks the next one to bf16 while it works on
// this one (with HALVES 2, four more waves do the same with every other tile, and the two sums are joined in LDS), into the order in
// which the products of 32 x 32 x 16 take it: fragments of 32 x 16 values, 16 bytes a lane. With
// i = lane & 31 and g = lane >> 5, K's fragment s has slot i, channels 16 s + 8 g .. + 7; the scores of row i and slots
// (r & 3) + 8 (r >> 2) + 4 g, r < 16, come out in the lane, which is how the second product takes the probabilities: of V's
// fragments 2 d and 2 d + 1, channel 32 d + i, entries r < 8 and r >= 8. The places are exchanged (XOR of the low three bits of a
// lane's place) so that the writes of unpacking and the reads of the products do not meet in a bank: of K's fragment s by g and
// 2 (s & 3), of V's by 4 g and d & 3.
//
// Bound by issuing instructions: 2 x 1024 tokens of 32 query heads over 8 of 128, lengths up to 8192 and 6000 positions in sight, bf16:
// 243 us between other calls, 252 in a row of forty, 473 and 457 TFLOP/s of scores and output (the output's products are done twice,
// for the probabilities' two parts; 68 % of all cycles issue something, the matrix units are busy for 28 %). With one part,
// probabilities held to 8 bits, 13 % less with four waves, and an error of 2.0e-3 instead of 1.7e-3 of bf16 outputs: not taken.
// fp32 and fp16 rows of 128 channels do not fit the registers whole (40 to 48 of them go to memory and back, one of fp16): 2 x 1024
// tokens over 8192 positions each take 695 and 537 us where bf16 takes 492.
template <int DH>
struct Unpacked {
    static constexpr int k = 64 * DH, bytes = 2 * k;
    __device__ static __forceinline__ int k_lane(int i, int g) { return 16 * ((i + 32 * g) ^ g); }
    __device__ static __forceinline__ int v_lane(int i, int g) { return k + 16 * ((i + 32 * g) ^ (4 * g)); }
    __device__ static __forceinline__ int k_at(int s, int lane) { return s * 1024 + (lane ^ (32 * (s & 3))); }
    __device__ static __forceinline__ int v_at(int d, int half, int lane) { return (2 * d + half) * 1024 + (lane ^ (16 * (d & 3))); }
};
constexpr int kManyRows = 128;
// Scores as powers of two. The running maximum is a rounded product, from which the others may differ by half its step before they are
// rounded: below kFar 2^-5, in every term of the row alike, from 2^33 on more than a power can hold. A row whose maximum is so far
// from zero is gone over again (as for NaN, below) with scores rounded as the maximum was, so that none is above it.
constexpr float kFar = 1 << 20;

template <int DH, class T, int HALVES>
__global__ __launch_bounds__(256 * HALVES, 2) void kv_attention_chunk_kernel(KvAttnArgs a, int row_tiles, int chunk_tiles) {
    using W = Width<DH>;
    using Tile = KvTile<DH>;
    using U = Unpacked<DH>;
    constexpr int QT = Terms<T>::q, PT = Terms<T>::p, KF = DH / 16, ND = DH / 32, o_raw = 2 * U::bytes, per_half = o_raw + 3 * Tile::bytes;
    constexpr int o_join = HALVES > 1 ? 4 * 16 * ND * 64 * 4 : 0;  // four waves' sums, then their maxima and sums of probabilities
    __shared__ __align__(16) uint8_t both[std::max(HALVES * per_half, o_join + 4 * 32 * 8)];
    const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5;
    const int half = HALVES > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0, tid = threadIdx.x - 256 * half;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint8_t* smem = both + half * per_half;
    const int unit = blockIdx.x;
    const int pair = unit / row_tiles, rt = unit - pair * row_tiles;
    const int s = pair / a.c.heads, h = pair - s * a.c.heads;
    const SeqSpan q = seq_span(a.pos, a.counts, s, a.T);
    const int ring = a.c.cap - a.c.sinks, sinks = a.c.sinks;
    const int t_lo = rt * kManyRows / a.group;
    if (t_lo >= q.count) return;
    const int t_hi = min((rt * kManyRows + kManyRows - 1) / a.group, q.count - 1);
    Seen seen;
    seen.sinks = sinks; seen.ring = ring; seen.window = a.window;
    seen.last = q.end - 1;
    seen.newest = seen.last >= sinks ? kv_slot(seen.last, sinks, ring) : -1;
    seen.lo_at = q.pos + t_lo;
    seen.hi_at = q.pos + t_hi;
    const Tiles tl = tiles_of(seen, a.c.cap);
    const int n_tiles = tl.count();
    // (four waves have their rows to themselves: only eight are given a chunk of the tiles)
    const int o0 = HALVES > 1 ? blockIdx.y * chunk_tiles : 0, o1 = HALVES > 1 ? min(n_tiles, o0 + chunk_tiles) : n_tiles;
    if (HALVES > 1 && blockIdx.y && o0 >= n_tiles) return;

    // loads of a tile: wave w has its w'th KiB, and one wave the scales
    constexpr int scale_wave = W::KS & 3;
    const size_t plane = (size_t)pair * a.c.cap;
    const uint32_t raw0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)(smem + o_raw);
    const int code_at = 1024 * wave + 16 * lane, scales_from = min(4 * (W::NB == 3 ? lane : lane & (16 * W::NB - 1)), 64 * W::NB - 4);
    const uint8_t* codes = code_at < Tile::half ? a.c.k + plane * Tile::row + code_at : a.c.v + plane * Tile::row + code_at - Tile::half;
    const uint8_t* scales = scales_from < 32 * W::NB ? a.c.ks + plane * W::NB + scales_from : a.c.vs + plane * W::NB + scales_from - 32 * W::NB;
    auto fetch = [&](int o, int slot) {
        const size_t j0 = tl.at(o) * kTile;
        if (wave < W::KS) lds_load16(codes + j0 * Tile::row, raw0 + slot * Tile::bytes + 1024 * wave);
        if (wave == scale_wave) lds_load4(scales + j0 * W::NB, raw0 + slot * Tile::bytes + Tile::o_scales);
    };
    // Unpacks a tile. Neighbouring lanes take neighbouring words of a row, of K a word, of V those of two slots; where they come from
    // and go to is found once.
    constexpr int words = DH / 8, NK = (32 * words + 255) / 256, NV = (16 * words + 255) / 256;
    int k_to[NK], v_from[NV], v_scale[NV], v_slot[NV], v_to[NV];
#pragma unroll
    for (int x = 0; x < NK; x++) {
        const int n = tid + 256 * x, j = n / words, wd = n % words;
        k_to[x] = U::k_at(wd / 2, U::k_lane(j, wd & 1));
    }
#pragma unroll
    for (int x = 0; x < NV; x++) {
        const int n = tid + 256 * x, j = n / words * 2, wd = n % words;
        v_from[x] = Tile::half + j * Tile::row + 4 * wd;
        v_scale[x] = Tile::o_scales + (32 + j) * W::NB + wd / 4;
        v_slot[x] = j;
        v_to[x] = U::v_at(wd / 4, j >> 4, U::v_lane(8 * (wd & 3), (j >> 2) & 1)) + 2 * ((j & 3) + (j >> 3 & 1) * 4);
    }
    auto unpack = [&](auto careful, int raw, int buf, int j0, bool held) {
        const uint8_t* p = smem + o_raw + raw * Tile::bytes;
        uint8_t* out = smem + buf * U::bytes;
#pragma unroll
        for (int x = 0; x < NK; x++) {
            if (32 * words % 256 && tid + 256 * x >= 32 * words) break;
            const int n = tid + 256 * x;  // (words and scales lie in the lanes' order)
            const uint32_t w = *(const uint32_t*)(p + 4 * n);
            const float sc = mx4_scale(p[Tile::o_scales + n / 4]);
            u32x4 y;
#pragma unroll
            for (int b = 0; b < 4; b++) y[b] = unpack2(w, sc, b);
            *(u32x4*)(out + k_to[x]) = y;
        }
#pragma unroll
        for (int x = 0; x < NV; x++) {
            if (16 * words % 256 && tid + 256 * x >= 16 * words) break;
            uint32_t w[2], sb[2];
#pragma unroll
            for (int y = 0; y < 2; y++) {
                w[y] = *(const uint32_t*)(p + v_from[x] + y * Tile::row);
                sb[y] = p[v_scale[x] + y * W::NB];
            }
            if (decltype(careful)::value || !held) {
                asm volatile("");
#pragma unroll
                for (int y = 0; y < 2; y++)
                    if (!seen.holds(j0 + v_slot[x] + y) || (decltype(careful)::value && sb[y] > 252u)) w[y] = sb[y] = 0;
            }
            const float s0 = mx4_scale(sb[0]), s1 = mx4_scale(sb[1]);
#pragma unroll
            for (int b = 0; b < 4; b++) {
                // channels 8 wd + 2 b and the next
                const uint32_t y0 = unpack2(w[0], s0, b), y1 = unpack2(w[1], s1, b);
                *(uint32_t*)(out + (v_to[x] ^ (32 * b))) = __builtin_amdgcn_perm(y1, y0, 0x05040100u);
                *(uint32_t*)(out + (v_to[x] ^ (32 * b + 16))) = __builtin_amdgcn_perm(y1, y0, 0x07060302u);
            }
        }
    };

    // this lane's row
    const int row = rt * kManyRows + wave * 32 + i, t = row / a.group, head = h * a.group + (row - t * a.group);
    const bool there = t < q.count;
    // its position and the last one behind its window; the wave's first and last positions
    const int at = q.pos + t, low = a.window > 0 ? at - a.window : INT_MIN;
    const int r0 = rt * kManyRows + wave * 32, lo = q.pos + r0 / a.group, hi = min(q.pos + (r0 + 31) / a.group, q.pos + q.count - 1);
    // the factor's sign, or zero, goes to the query, so that the largest product is the largest score
    const float sign = a.scale < 0.0f ? -1.0f : a.scale == 0.0f ? 0.0f : 1.0f, scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
    v8bf qf[KF][QT];
    {
        const T* p = (const T*)a.q.data + s * a.q.seq + t * a.q.token + head * a.q.head + 8 * g;
#pragma unroll
        for (int x = 0; x < KF; x++) {
            float y[8] = {};
            if (there) real_load8<T>(p + 16 * x, 8, y);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] *= sign;
            split_bf16<QT>(y, qf[x]);
        }
    }
    v16f acc[ND];
    float m, l;
    uint32_t nan_blocks;

    auto barrier = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
    // run: the position of the tile's first slot, where its slots hold 32 positions in a row
    auto work = [&](auto careful, int buf, int j0, int run) {
        if (lo > hi || (run >= 0 && (run > hi || (a.window > 0 && run + 31 <= lo - a.window)))) return;  // no row sees it
        const uint8_t* p = smem + buf * U::bytes;
        int k_lane = U::k_lane(i, g), v_lane = U::v_lane(i, g);
        asm volatile("" : "+v"(k_lane), "+v"(v_lane));
        v16f d = {};
#pragma unroll
        for (int x = 0; x < KF; x++) {
            const v8bf kf = *(const v8bf*)(p + U::k_at(x, k_lane));
#pragma unroll
            for (int n = QT - 1; n >= 0; n--) d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[x][n], d, 0, 0, 0);
        }
        const bool whole = run >= 0 && run + 31 <= lo && (a.window <= 0 || run > hi - a.window);
        if (!whole) {
            asm volatile("");
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int j = j0 + (r & 3) + 8 * (r >> 2) + 4 * g;
                const bool v = seen.sees(j, at, low);
                d[r] = v ? d[r] : -INFINITY;
                if (decltype(careful)::value && v)
                    for (int b = 0; b < W::NB; b++)
                        if (a.c.vs[(plane + j) * W::NB + b] > 252u) nan_blocks |= 1u << b;
            }
        }
        float mt = d[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mt = fmaxf(mt, d[r]);
        // (in units of the score's power of two; a row that sees nothing here stays as it is)
        mt = mt == -INFINITY ? -INFINITY : mt * scale;
        if (__any(mt > m)) {  // rare after the first tiles
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
            const float mn = fmaxf(m, fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])));
            const float al = __builtin_amdgcn_exp2f(mn == -INFINITY ? 0.0f : m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int x = 0; x < ND; x++) acc[x] *= al;
        }
        const float mu = m == -INFINITY ? 0.0f : m;
        float pr[16];
#pragma unroll
        for (int r = 0; r < 16; r++)
            pr[r] = __builtin_amdgcn_exp2f(decltype(careful)::value && fabsf(mu) >= kFar ? d[r] * scale - mu : fmaf(d[r], scale, -mu));
        float sum[4];
#pragma unroll
        for (int r = 0; r < 4; r++) sum[r] = (pr[r] + pr[4 + r]) + (pr[8 + r] + pr[12 + r]);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        v8bf pf[2][PT];
        split_bf16<PT>(pr, pf[0]);
        split_bf16<PT>(pr + 8, pf[1]);
#pragma unroll
        for (int x = 0; x < ND; x++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const v8bf vf = *(const v8bf*)(p + U::v_at(x, hf, v_lane));
#pragma unroll
                for (int n = PT - 1; n >= 0; n--) acc[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[hf][n], acc[x], 0, 0, 0);
            }
    };
    auto sweep = [&](auto careful) {
#pragma unroll
        for (int x = 0; x < ND; x++) acc[x] = v16f{};
        m = -INFINITY;
        l = 0.0f;
        nan_blocks = 0;
        if (o1 <= o0) return;
        const int first = o0 + half, n = (o1 - first + HALVES - 1) / HALVES;  // this half's tiles; the other's may be one more
        for (int x = 0; x < min(n, 3); x++) fetch(first + HALVES * x, x);
        vm_wait<0>();
        barrier();
        int j0 = tl.at(min(first, o1 - 1)) * kTile, run = seen.run(j0);
        if (HALVES == 1 || n > 0) unpack(careful, 0, 0, j0, run >= 0);
        int raw = 0;  // of tile x
        for (int x = 0; x < (o1 - o0 + HALVES - 1) / HALVES; x++) {
            // tile x is unpacked, tile x + 1 has landed; tile x's raw place and the other unpacked one are free
            barrier();
            if (HALVES > 1 && x >= n) break;  // (the last time around)
            if (x + 3 < n) fetch(first + HALVES * (x + 3), raw);
            raw = raw == 2 ? 0 : raw + 1;
            const int j1 = tl.at(first + HALVES * min(x + 1, n - 1)) * kTile, run1 = seen.run(j1);
            if (x + 1 < n) unpack(careful, raw, (x + 1) & 1, j1, run1 >= 0);
            // (the careful form asks for every slot of every tile)
            work(careful, x & 1, j0, decltype(careful)::value ? -1 : run);
            j0 = j1;
            run = run1;
            // all but this step's loads have landed
            if (x + 3 >= n) vm_wait<0>();
            else if (W::KS == 4 && wave == scale_wave) vm_wait<2>();
            else vm_wait<1>();
        }
    };
    sweep(std::false_type());
    {
        // A NaN among the sums: it may come from a value that the row does not see. Or scores far from zero.
        float bad = 0.0f;
#pragma unroll
        for (int x = 0; x < ND; x++)
#pragma unroll
            for (int r = 0; r < 16; r++) bad += acc[x][r] * 0.0f;
        if (__syncthreads_or(bad != 0.0f || (m != -INFINITY && fabsf(m) >= kFar))) {
            sweep(std::true_type());
            nan_blocks |= __shfl_xor(nan_blocks, 32, 64);
#pragma unroll
            for (int x = 0; x < ND; x++)
                if (nan_blocks >> x & 1)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[x][r] = NAN;
        }
    }
    float total = l + __shfl_xor(l, 32, 64);
    if constexpr (HALVES > 1) {
        // the halves' sums, at the larger maximum
        float* s_o = (float*)both + wave * 16 * ND * 64 + lane;
        float* s_ml = (float*)(both + o_join) + (wave * 32 + i) * 2;
        __syncthreads();
        if (half) {
#pragma unroll
            for (int x = 0; x < ND; x++)
#pragma unroll
                for (int r = 0; r < 16; r++) s_o[(16 * x + r) * 64] = acc[x][r];
            if (g == 0) {
                s_ml[0] = m;
                s_ml[1] = total;
            }
        }
        __syncthreads();
        if (half) return;
        const float m1 = s_ml[0], top = fmaxf(m, m1), tu = top == -INFINITY ? 0.0f : top;
        const float f0 = __builtin_amdgcn_exp2f(m - tu), f1 = __builtin_amdgcn_exp2f(m1 - tu);
        m = top;
        total = total * f0 + s_ml[1] * f1;
#pragma unroll
        for (int x = 0; x < ND; x++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[x][r] = acc[x][r] * f0 + s_o[(16 * x + r) * 64] * f1;
    }
    if (!there) return;
    // lane (i, g): row i, channels 32 x + 8 r + 4 g .. + 3
    if (HALVES > 1 && n_tiles > chunk_tiles) {
        float* part = a.ws + (((size_t)blockIdx.y * gridDim.x + unit) * kManyRows + wave * 32 + i) * kPart<DH>;
#pragma unroll
        for (int x = 0; x < ND; x++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *(v4f*)(part + 32 * x + 8 * r + 4 * g) = v4f{acc[x][4 * r], acc[x][4 * r + 1], acc[x][4 * r + 2], acc[x][4 * r + 3]};
        if (g == 0) {
            part[DH] = m;
            part[DH + 1] = total;
        }
    } else {
        const float f = total == 0.0f ? 0.0f : 1.0f / total;
        T* out = (T*)a.out.data + s * a.out.seq + t * a.out.token + head * a.out.head;
#pragma unroll
        for (int x = 0; x < ND; x++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                real_store4(out + 32 * x + 8 * r + 4 * g, v4f{acc[x][4 * r], acc[x][4 * r + 1], acc[x][4 * r + 2], acc[x][4 * r + 3]} * f, 4);
    }
}

// How a call is divided: `per` rows a unit (a row tile of one head, or all rows of hb heads), `waves` sharing a unit's tiles, `chunks`
// workgroups a unit.
struct AttnPlan {
    bool many;  // kv_attention_chunk_kernel
    int per, hb, row_tiles, units, waves, chunk_tiles, chunks;
};
AttnPlan attn_plan(const KvAttnArgs& a) {
    AttnPlan p;
    const int rows = a.T * a.group, most = a.c.dh == 32 ? 8 : a.c.dh == 64 ? 4 : 2;
    // (32 conversations of 4096 positions, 32 heads of 128 over 8, bf16, 24 and 32 rows a head: 90 and 120 us eight rows a wave, 129
    // in both with many; 64 of 2048, fp32 heads of 64: 62 and 88, 124 in both)
    p.many = rows > 32;
    // heads a wave takes together: as many as give it 8 rows or fewer
    p.hb = rows * most <= kRows && a.c.heads % most == 0 ? most : rows * 2 <= kRows && a.c.heads % 2 == 0 ? 2 : 1;
    p.per = p.many ? kManyRows : kRows;
    p.row_tiles = (rows - 1) / p.per + 1;  // (rows are fewer than 2^31, but not by a tile)
    p.units = a.c.n * (a.c.heads / p.hb) * p.row_tiles;
    // tiles that a row tile can see, at most: the sinks', and the window's (or the ring's), with the ends of three runs
    const long long span = a.window > 0 ? std::min<long long>((long long)a.window + p.per / a.group + 1, a.c.cap) : a.c.cap;
    const int tiles = (int)std::min<long long>((span + kTile - 1) / kTile + (a.c.sinks + kTile - 1) / kTile + 2, a.c.cap / kTile);
    // Many rows, eight waves, four for every other tile, where no more than two workgroups of four a CU would be there: they all
    // start at once, and nothing takes the place of one that ends early. The lengths are not known here: unequal ones gain, equal ones
    // that fill the card lose a few percent (us, four waves and eight, in rows of forty, bf16 heads of 128 but where said: 2 x 1024
    // tokens, 512 workgroups, over up to 8192 positions 360 and 298, over 8192 each 452 and 492, the same in fp16 497 and 537, in fp32
    // 780 and 695; 16 x 256 tokens over up to 4096, fp16 heads of 64, 256 workgroups 148 and 102; 4 x 512 over 4096 each, fp32 heads of
    // 64, 256 workgroups 228 and 240; 64 tokens over 2048, 4 workgroups 94 and 28; and where more are waiting, 8 x 512 tokens over 4096,
    // 1024 workgroups 509 and 523; with two tiles to share, 256 x 64 tokens, heads of 64, 36 and 58)
    p.waves = p.many ? (p.units <= 512 && tiles >= 16 ? 8 : 4) : tiles <= 4 ? 1 : 4;
    p.chunk_tiles = tiles;
    if (p.many ? p.waves == 8 : p.waves > 1) {
        // Two workgroups a CU (one of eight waves), each with four tiles a wave at least (sixteen a workgroup of many rows). More,
        // smaller chunks cost more at their ends than they even out (256 conversations, their window in one chunk or two: 29 or
        // 38 us). Many rows on four waves have more workgroups than that, or few tiles.
        const int want = std::max(1, (p.waves == 8 ? 256 : 512) / p.units);
        p.chunk_tiles = std::max(16, (tiles + want - 1) / want);
    }
    p.chunks = std::max(1, (tiles + p.chunk_tiles - 1) / p.chunk_tiles);
    return p;
}

template <int DH, class T>
hipError_t launch_join(const KvAttnArgs& a, const AttnPlan& p, hipStream_t s) {
    if (p.chunks > 1) {
        const int cols = p.hb > 1 ? p.hb * a.T * a.group : std::min(p.per, a.T * a.group);
        hipLaunchKernelGGL((kv_attention_join_kernel<DH, T>), dim3(p.units, (cols + 3) / 4), dim3(256), 0, s, a, p.per, p.hb, p.row_tiles,
                           p.chunk_tiles);
    }
    return hipGetLastError();
}

template <int DH, class T, int HB>
hipError_t launch_rows_attention(const KvAttnArgs& a, const AttnPlan& p, hipStream_t s) {
    if (p.waves == 1) {
        hipLaunchKernelGGL((kv_attention_rows_kernel<DH, T, HB, 1>), dim3((p.units + 3) / 4), dim3(256), 0, s, a, p.row_tiles, p.chunk_tiles);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((kv_attention_rows_kernel<DH, T, HB, 4>), dim3(p.units, p.chunks), dim3(256), 0, s, a, p.row_tiles, p.chunk_tiles);
    return launch_join<DH, T>(a, p, s);
}

}  // namespace

bool kv_head_width(int dh) { return dh == 32 || dh == 64 || dh == 96 || dh == 128; }

hipError_t launch_kv_write(const KvRowsArgs& a, hipStream_t s) { return launch_rows<false>(a, s); }
hipError_t launch_kv_read(const KvRowsArgs& a, hipStream_t s) { return launch_rows<true>(a, s); }

size_t kv_attention_ws_bytes(const KvAttnArgs& a) {
    const AttnPlan p = attn_plan(a);
    return p.chunks > 1 ? (size_t)p.chunks * p.units * p.per * (a.c.dh + 4) * 4 : 0;
}

bool kv_attention_fits(const KvAttnArgs& a) {
    const AttnPlan p = attn_plan(a);
    return (p.waves == 1 ? (p.units + 3) / 4 : p.units) < 1 << 24;  // a launch's 2^32 lanes
}

hipError_t launch_kv_attention(const KvAttnArgs& a, hipStream_t s) {
    const AttnPlan p = attn_plan(a);
    return by_width(a.c.dh, [&](auto w) {
        constexpr int DH = decltype(w)::value, most = DH == 32 ? 8 : DH == 64 ? 4 : 2;
        return by_real(a.type, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (p.many) {
                if (p.waves == 4) {
                    hipLaunchKernelGGL((kv_attention_chunk_kernel<DH, T, 1>), dim3(p.units), dim3(256), 0, s, a, p.row_tiles, p.chunk_tiles);
                    return hipGetLastError();
                }
                hipLaunchKernelGGL((kv_attention_chunk_kernel<DH, T, 2>), dim3(p.units, p.chunks), dim3(512), 0, s, a, p.row_tiles, p.chunk_tiles);
                return launch_join<DH, T>(a, p, s);
            }
            if (p.hb == most) return launch_rows_attention<DH, T, most>(a, p, s);
            if constexpr (most > 2)
                if (p.hb == 2) return launch_rows_attention<DH, T, 2>(a, p, s);
            return launch_rows_attention<DH, T, 1>(a, p, s);
        });
    });
}

}  // namespace mg
