// Device code that the kernels over 4-bit caches share: where a sequence's positions are, the tiles that a call reads, a tile's layout in LDS and
// its unpacking, masks.
#pragma once

#include <algorithm>
#include <climits>

#include "common.hpp"
#include "mx4.hpp"
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

template <class F>
auto by_width(int dh, F&& f) {
    switch (dh) {
        case 32: return f(std::integral_constant<int, 32>());
        case 64: return f(std::integral_constant<int, 64>());
        case 96: return f(std::integral_constant<int, 96>());
        default: return f(std::integral_constant<int, 128>());
    }
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

}  // namespace
}  // namespace mg
