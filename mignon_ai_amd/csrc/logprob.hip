// Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits.
//
// With m the largest logit of a row, S = sum e^(x - m) and X = sum (x - m) e^(x - m): log p(t) = (x_t - m) - log S, and the entropy is
// log S - X / S. One pass over the row: a lane keeps its own running maximum and sums, at 2^(x c - r) with c = log2 e and r = m c rounded,
// one fused operation a power; sums at one r are put at another by 2^(r - r'), and at the end r's rounding, d = m c - r, is taken out
// of log S (it cancels in the entropy).
//
// The k likeliest: a wave looks at tiles of 2048 logits, 32 a lane. The k-th of the lanes' maxima is at most the k-th of the tile, so only what
// reaches it can be among the k: in ordinary rows few more than k. Where the k-th is met by more than there is room for (many equal logits, as
// in masked rows), numbers and ids together, one 64-bit key, no two alike, bound it: at most k lanes reach the bound then, with 32 logits
// each. Later tiles are held to the bound so far, and one whose lanes' maxima all fail it (most do) costs nothing more. Candidates are put in
// order by counting, for each, those above it. A wave does all that by itself; up to four share a row, and meet at its end.
//
// Bound by memory without alternatives (16384 rows of 8192 fp32 logits, 537 MB: 85 to 90 us, 6.1 TB/s; 512 of 100003 bf16 23.7, 4.3 TB/s), by the
// first tiles' candidates with them (the same 512 with 1, 5, 16 and 64 alternatives: 37 43 52 93; all four waves agreeing on a bound tile by
// tile took 54 60 66 118), by latency for few rows (16 of 8192 with 5: 7.6; one of 131072 with 20: 12 and 4.7 to join 16 segments).
//
// What this does badly: rows whose first tile bounds nothing. The numbers' bound is found on a wave's first tile alone; where that is forbidden
// throughout (-infinity), the first tile with numbers is taken whole. Up to 55 alternatives that overflows the room, and the exact bound
// follows; from 56 on the room holds it, and one wave puts some 2100 candidates in order by counting. The same 512 rows with the first third of
// the ids forbidden (a third at random costs nothing): 66 us with 1 alternative, 83 with 16, 1940 with 64; all logits equal 71, 77, 966;
// every tile above the one before 140, 227, 11270.
#include "logprob.hpp"

#include <algorithm>

#include "common.hpp"
#include "mx4_device.hpp"

namespace mg {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kHuge = 0x1p20f;  // from here on a rounding of m c is more than 2^-4: such rows are gone over again, by differences
constexpr float kNothing = -200.0f;  // 2^-200 is 0: stands for -infinity where that would be multiplied with 0

// A logit and its id as one number: larger is likelier, the lowest id first among equals, -0 as 0, NaN below all. Never 0.
__device__ __forceinline__ uint64_t top_key(float x, int id) {
    const uint32_t b = __float_as_uint(x + 0.0f), o = x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)o << 32 | (uint32_t)~id;
}
__device__ __forceinline__ int key_id(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t o = key >> 32;
    return o == 0 ? NAN : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// What a segment of a row gave: its maximum, S and X (in powers of two) at it; then its k largest keys.
struct Part {
    float m, S, X, pad;
};
__host__ __device__ constexpr size_t part_bytes(int k) { return sizeof(Part) + 8 * (size_t)k; }

// Eight neighbouring logits as they lie in memory.
template <class T>
struct Raw8 {
    using R = typename Raw16<sizeof(T)>::type;
    R r[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p, int left) {
        if (left >= 8) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) r[i] = ((const R*)p)[i];
        } else {
            T t[8];
#pragma unroll
            for (int e = 0; e < 8; e++) t[e] = e < left ? p[e] : (T)-INFINITY;
            __builtin_memcpy(r, t, sizeof(t));
        }
    }
    __device__ __forceinline__ void get(float x[8]) const {
        T t[8];
        __builtin_memcpy(t, r, sizeof(t));
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)t[e];
    }
};

// Between lanes of a wave, through LDS.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

constexpr int kTile = 2048;  // logits of a wave's tile
// A wave's candidates, in LDS.
struct Top {
    uint64_t* keys;   // room
    uint64_t* best;   // the k best in order; lanes' keys
    int* count;
    int k, room, l;
    uint64_t bound = 1;
    static __host__ __device__ int room_of(int k) { return 32 * k + 256; }
    static __host__ __device__ int bytes(int k) { return k ? 8 * (room_of(k) + 64) + 16 : 0; }
    __device__ __forceinline__ Top(uint8_t* at, int k_, int l_) : k(k_), room(room_of(k_)), l(l_) {
        keys = (uint64_t*)at;
        best = keys + room;
        count = (int*)(best + 64);
    }
    // Raises the bound to the k-th largest of the lanes' maxima, or, for many, of those of their halves (of 64 maxima the 64th is met by 300
    // of 2048 logits, of 128 by 90), by their numbers alone. A lane without numbers has none.
    static __device__ __forceinline__ uint32_t number(float m) { return m > -INFINITY ? (uint32_t)(top_key(m, 0) >> 32) : 0u; }
    __device__ __forceinline__ void tighten(float m0, float m1) {
        uint32_t h0 = number(m0), h1 = number(m1), kth;
        if (k <= 16) {
            h0 = max(h0, h1);
            int above = 0;
#pragma unroll
            for (int j = 0; j < 64; j++) above += (uint32_t)__builtin_amdgcn_readlane((int)h0, j) > h0;
            kth = wave_min(above < k ? h0 : ~0u);
        } else {
            int a0 = 0, a1 = 0;
#pragma unroll 16
            for (int j = 0; j < 64; j++) {
                const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)h0, j), y = (uint32_t)__builtin_amdgcn_readlane((int)h1, j);
                a0 += (x > h0) + (y > h0);
                a1 += (x > h1) + (y > h1);
            }
            kth = wave_min(min(a0 < k ? h0 : ~0u, a1 < k ? h1 : ~0u));
        }
        const uint64_t key = (uint64_t)kth << 32;
        bound = key > bound ? key : bound;
    }
    __device__ void tighten_exactly(uint64_t mine) {
        best[l] = mine;
        wave_fence();
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < 64; j++) above += best[j] > mine || (best[j] == mine && j < l);  // (lanes without logits are alike)
        const uint64_t who = __ballot(above == k - 1);
        const uint64_t kth = __shfl((unsigned long long)mine, __ffsll((unsigned long long)who) - 1, 64);
        bound = kth > bound ? kth : bound;
        wave_fence();
    }
    __device__ __forceinline__ void push(uint64_t key) {
        if (key < bound) return;
        const int at = atomicAdd(count, 1);
        if (at < room) keys[at] = key;
    }
    // Leaves the k largest of n candidates, in order, and raises the bound to the last of them.
    __device__ int select(int n) {
        for (int c = l; c < n; c += 64) {
            const uint64_t key = keys[c];
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < n; j++) above += keys[j] > key;
            if (above < k) best[above] = key;
        }
        wave_fence();
        const int left = min(n, k);
        if (l < left) keys[l] = best[l];
        if (l == 0) *count = left;
        if (left == k) bound = best[k - 1] > bound ? best[k - 1] : bound;
        wave_fence();
        return left;
    }
};

// WAVES waves take a segment of a row, tile by tile in turns, each wave's next tile loaded while it works on one.
template <class T, int WAVES>
__global__ __launch_bounds__(256) void logprob_kernel(LogprobArgs a, int splits, int segment) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_part[3][4];
    __shared__ uint64_t s_best[kMaxTop];
    constexpr int lanes = 64 * WAVES, teams = 4 / WAVES;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), team = wave / WAVES, w = wave % WAVES;
    const int lane = threadIdx.x & 63, l = 64 * w + lane;
    const long long unit = (long long)blockIdx.x * teams + team;
    if (unit >= (long long)a.n * splits) return;  // (a wave by itself, or all four)
    const long long r = splits == 1 ? unit : unit / splits;
    const int part = (int)(unit - r * splits), from = part * segment, to = min(a.V, from + segment);
    const T* x = (const T*)a.x + r * a.ld;
    Top top(smem + wave * Top::bytes(a.k), a.k, lane);

    Raw8<T> next[4];
    auto fetch = [&](int v0) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int v = v0 + (j * 64 + lane) * 8;
            next[j].load(x + v, to - v);
        }
    };
    const int begin = from + kTile * w;
    if (begin < to) fetch(begin);
    // a lane's target
    int target = -1;
    float x_t = NAN;
    if (splits == 1 && l < a.m) {
        target = a.targets[r * a.m + l];
        if (target >= 0 && target < a.V) x_t = (float)x[target];
    }
    float m = -INFINITY, at = 0.0f, S = 0.0f, X = 0.0f;  // at: r
    int n = 0;                                           // candidates
    if (a.k) {
        if (lane == 0) *top.count = 0;
        wave_fence();
    }
    for (int v0 = begin; v0 < to; v0 += kTile * WAVES) {
        float y[32];
#pragma unroll
        for (int j = 0; j < 4; j++) next[j].get(y + 8 * j);
        if (v0 + kTile * WAVES < to) fetch(v0 + kTile * WAVES);
        float m0 = y[0], m1 = y[16];
#pragma unroll
        for (int e = 1; e < 16; e++) {
            m0 = fmaxf(m0, y[e]);
            m1 = fmaxf(m1, y[16 + e]);
        }
        const float mt = fmaxf(m0, m1);
        if (__any(mt > m)) {
            const float mn = fmaxf(m, mt), an = fmaxf(mn, -kHuge) * kLog2e, f = __builtin_amdgcn_exp2f(at - an);
            // (a lane with nothing above -kHuge adds nothing to a row that has more; S 0: there is no reference to leave)
            X = S == 0.0f ? 0.0f : (X + S * (at - an)) * f;
            S = S == 0.0f ? 0.0f : S * f;
            m = mn;
            at = an;
        }
        float s4[4] = {}, x4[4] = {};
#pragma unroll
        for (int e = 0; e < 32; e++) {
            const float d = fmaf(y[e], kLog2e, -at), p = __builtin_amdgcn_exp2f(d);
            s4[e & 3] += p;
            x4[e & 3] = fmaf(p, fmaxf(d, kNothing), x4[e & 3]);
        }
        S += (s4[0] + s4[1]) + (s4[2] + s4[3]);
        X += (x4[0] + x4[1]) + (x4[2] + x4[3]);
        if (!a.k) continue;
        const bool first = v0 == begin;
        if (!first && !__any((top.bound >> 32) == 0 || mt >= key_value(top.bound))) continue;
        const auto id_of = [&](int e) { return v0 + ((e >> 3) * 64 + lane) * 8 + (e & 7); };
        // the lane's first largest logit (what is not there, behind the end, is -infinity and comes last)
        const auto largest = [&] {
            int at = 0;
#pragma unroll
            for (int e = 31; e >= 0; e--) at = y[e] == mt ? e : at;
            uint64_t key = id_of(at) < to ? top_key(mt, id_of(at)) : 0;
            if (!(mt > -INFINITY)) {
                // nothing but -infinity, NaN, and what is not there
                asm volatile("");
                key = 0;
#pragma unroll
                for (int e = 31; e >= 0; e--) {
                    const uint64_t other = id_of(e) < to ? top_key(y[e], id_of(e)) : 0;
                    key = other > key ? other : key;
                }
            }
            return key;
        };
        const auto push = [&] {
            // (NaN is not below anything: its key decides)
            const float low = (top.bound >> 32) == 0 ? -INFINITY : key_value(top.bound);
#pragma unroll
            for (int e = 0; e < 32; e++)
                if (!(y[e] < low) && id_of(e) < to) top.push(top_key(y[e], id_of(e)));
            wave_fence();
            return *top.count;
        };
        if (first) top.tighten(m0, m1);
        int now = push();
        if (now > top.room) {
            // more than there is room for reach the bound so far: once more, with the tile's own
            wave_fence();
            if (lane == 0) *top.count = n;
            wave_fence();
            n = top.select(n);
            top.tighten_exactly(largest());
            now = push();
        }
        n = now;
        wave_fence();
        if (n > a.k + a.k / 2 + 8) n = top.select(n);
    }
    // the row's: lanes' sums at the largest maximum
    float most = wave_max(m);
    if constexpr (WAVES > 1) {
        if (lane == 0) s_part[0][w] = most;
        __syncthreads();
        most = fmaxf(fmaxf(s_part[0][0], s_part[0][1]), fmaxf(s_part[0][2], s_part[0][3]));
    }
    float ref = most == -INFINITY ? 0.0f : most * kLog2e, off = fmaf(most, kLog2e, -ref);
    if (fabsf(most) >= kHuge && most < INFINITY && most > -INFINITY) {
        S = X = ref = at = off = 0.0f;
        for (int v = from + l; v < to; v += lanes) {
            const float d = ((float)x[v] - most) * kLog2e, p = __builtin_amdgcn_exp2f(d);
            S += p;
            X = fmaf(p, fmaxf(d, kNothing), X);
        }
    }
    {
        const float f = __builtin_amdgcn_exp2f(at - ref);
        X = S == 0.0f ? 0.0f : (X + S * (at - ref)) * f;
        S = S == 0.0f ? 0.0f : S * f;
    }
    S = wave_sum(S);
    X = wave_sum(X);
    const uint64_t* best = top.best;
    if (a.k) n = top.select(n);
    if constexpr (WAVES > 1) {
        if (lane == 0) {
            s_part[1][w] = S;
            s_part[2][w] = X;
        }
        if (a.k && lane < a.k && lane >= n) top.keys[lane] = 0;
        __syncthreads();
        S = (s_part[1][0] + s_part[1][1]) + (s_part[1][2] + s_part[1][3]);
        X = (s_part[2][0] + s_part[2][1]) + (s_part[2][2] + s_part[2][3]);
        if (a.k) {
            // the waves' lists, in order each
            if (lane < a.k) {
                const uint64_t key = top.keys[lane];
                int above = lane;
                for (int o = 1; o < WAVES; o++) {
                    const uint64_t* other = (const uint64_t*)(smem + (w ^ o) * Top::bytes(a.k));
                    int lo = 0, hi = a.k;  // other[lo - 1] > key >= other[hi]
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        if (other[mid] > key) lo = mid + 1;
                        else hi = mid;
                    }
                    above += lo;
                }
                if (above < a.k && key) s_best[above] = key;
            }
            __syncthreads();
            n = min(a.k, to - from);
            best = s_best;
        }
    }
    if (splits > 1) {
        uint8_t* out = (uint8_t*)a.ws + unit * part_bytes(a.k);
        if (most == -INFINITY) off = 0.0f;
        if (l == 0) {
            const float f = __builtin_amdgcn_exp2f(-off);
            *(Part*)out = Part{most, S * f, (X - off * S) * f, 0.0f};
        }
        uint64_t* keys = (uint64_t*)(out + sizeof(Part));
        if (l < a.k) keys[l] = l < n ? best[l] : 0;  // (k is at most 64)
        return;
    }
    const float log_s = logf(S) - off * kLn2;
    if (a.entropy && l == 0) a.entropy[r] = logf(S) - X / S * kLn2;
    for (int j = l; j < a.m; j += lanes) {
        if (j != l) {
            target = a.targets[r * a.m + j];
            x_t = target >= 0 && target < a.V ? (float)x[target] : NAN;
        }
        a.logprob[r * a.m + j] = (x_t - most) - log_s;
    }
    if (l < a.k) {
        const uint64_t key = best[l];
        if (a.top_ids) a.top_ids[r * a.k + l] = key_id(key);
        if (a.top_logprob) a.top_logprob[r * a.k + l] = (key_value(key) - most) - log_s;
    }
}

// A row's segments (64 at most): sums at the largest maximum, and the k largest of their k largest keys each. The k-th of the lists' first keys is
// at most the k-th of all; few more than k reach it.
template <class T>
__global__ __launch_bounds__(256) void logprob_join_kernel(LogprobArgs a, int splits) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int l = threadIdx.x;
    const long long r = blockIdx.x;
    const T* x = (const T*)a.x + r * a.ld;
    const uint8_t* parts = (const uint8_t*)a.ws + r * splits * part_bytes(a.k);
    int target = -1;
    float x_t = NAN;
    if (l < a.m) {
        target = a.targets[r * a.m + l];
        if (target >= 0 && target < a.V) x_t = (float)x[target];
    }
    // (each wave for itself; at most 64 segments)
    const int w = l & 63;
    Part p = {-INFINITY, 0.0f, 0.0f, 0.0f};
    if (w < splits) p = *(const Part*)(parts + w * part_bytes(a.k));
    const float most = wave_max(p.m);
    {
        const float d = p.m == -INFINITY && p.S == 0.0f ? 0.0f : fmaxf((p.m - most) * kLog2e, kNothing), f = __builtin_amdgcn_exp2f(d);
        p.X = (p.X + p.S * d) * f;
        p.S *= f;
    }
    const float S = wave_sum(p.S), X = wave_sum(p.X), log_s = logf(S);
    if (a.entropy && l == 0) a.entropy[r] = log_s - X / S * kLn2;
    for (int j = l; j < a.m; j += 256) {
        if (j != l) {
            target = a.targets[r * a.m + j];
            x_t = target >= 0 && target < a.V ? (float)x[target] : NAN;
        }
        a.logprob[r * a.m + j] = (x_t - most) - log_s;
    }
    if (!a.k) return;
    uint64_t* keys = (uint64_t*)smem;
    __shared__ uint64_t s_best[kMaxTop], s_heads[192], s_low;
    __shared__ int s_count;
    if (l == 0) s_count = 0;
    // the k-th of the lists' first keys, some 2 k of them
    const int deep = min(a.k, (2 * a.k - 1) / splits + 1), heads = splits * deep;  // k to 2 k + 63
    uint64_t key = 0;
    if (l < heads) {
        const int s = l / deep;
        key = ((const uint64_t*)(parts + s * part_bytes(a.k) + sizeof(Part)))[l - s * deep];
        s_heads[l] = key;
    }
    __syncthreads();
    if (l < heads) {
        int above = 0;  // (0: no key, all alike)
#pragma unroll 16
        for (int j = 0; j < heads; j++) above += s_heads[j] > key || (s_heads[j] == key && j < l);
        if (above == a.k - 1) s_low = key;
    }
    __syncthreads();
    const uint64_t low = s_low;
    for (int c = l; c < splits * a.k; c += 256) {
        const int s = c / a.k;
        const uint64_t key = ((const uint64_t*)(parts + s * part_bytes(a.k) + sizeof(Part)))[c - s * a.k];
        if (key >= low && key) keys[atomicAdd(&s_count, 1)] = key;
    }
    __syncthreads();
    const int n = s_count;
    for (int c = l; c < n; c += 256) {
        const uint64_t key = keys[c];
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) above += keys[j] > key;
        if (above < a.k) s_best[above] = key;
    }
    __syncthreads();
    if (l < a.k) {
        const uint64_t key = s_best[l];
        if (a.top_ids) a.top_ids[r * a.k + l] = key_id(key);
        if (a.top_logprob) a.top_logprob[r * a.k + l] = (key_value(key) - most) - log_s;
    }
}

// A wave a row where rows are short, or so many that waves alone fill the chip (then each finds its first candidates once), four elsewhere; long
// rows in segments where there are fewer than 512. us, a wave a row and four: 16384 rows of 1000 bf16 17.8 and 52; of 2048 fp32 with 5
// alternatives 34 and 102, of 4096 53 and 108, of 8192 101 and 128, without 93 and 87; 4096 of 32768 with 5 105 and 100; 2048 of 8192 with 5
// 18.8 and 22, 1024 14.9 and 11.2; 64 of 4096 13.3 and 9.1. Segments for 512 workgroups and for 2048: 512 rows of 100003 bf16 without
// alternatives 22.6 and 26.4, with 16 50 and 63; 32 of 131072 19.6 and 19.4.
struct LogprobPlan {
    int waves, splits, segment;
};
LogprobPlan logprob_plan(const LogprobArgs& a) {
    LogprobPlan p;
    p.waves = a.V <= 2048 || (a.n >= 2048 && a.V <= (a.k ? 8192 : 4096)) ? 1 : 4;
    const int tile = kTile * p.waves, tiles = (a.V - 1) / tile + 1;
    const int want = std::min(64, std::max(1, std::min(tiles, 512 / std::max(a.n, 1))));
    p.segment = (tiles + want - 1) / want * tile;
    p.splits = (a.V - 1) / p.segment + 1;
    return p;
}

template <class T, int WAVES>
hipError_t launch_rows(const LogprobArgs& a, const LogprobPlan& p, hipStream_t s) {
    const long long units = (long long)a.n * p.splits;
    const int teams = 4 / WAVES;
    static std::atomic<uint64_t> allowed{0};
    if (const hipError_t e = allow_lds((const void*)logprob_kernel<T, WAVES>, 4 * Top::bytes(kMaxTop), allowed); e != hipSuccess) return e;
    hipLaunchKernelGGL((logprob_kernel<T, WAVES>), dim3((unsigned)((units + teams - 1) / teams)), dim3(256), 4 * Top::bytes(a.k), s, a,
                       p.splits, p.segment);
    return hipGetLastError();
}

}  // namespace

// (a launch's 2^32 lanes; a workgroup takes four rows of a wave each)
bool logprob_fits(const LogprobArgs& a) {
    const LogprobPlan p = logprob_plan(a);
    const int teams = 4 / p.waves;
    return ((long long)a.n * p.splits + teams - 1) / teams < 1 << 24;
}
size_t logprob_ws_bytes(const LogprobArgs& a) {
    const LogprobPlan p = logprob_plan(a);
    return p.splits > 1 ? (size_t)a.n * p.splits * part_bytes(a.k) : 0;
}

hipError_t launch_logprob(const LogprobArgs& a, hipStream_t s) {
    const LogprobPlan p = logprob_plan(a);
    return by_real(a.type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const hipError_t e = p.waves == 1 ? launch_rows<T, 1>(a, p, s) : launch_rows<T, 4>(a, p, s);
        if (e != hipSuccess || p.splits == 1) return e;
        hipLaunchKernelGGL((logprob_join_kernel<T>), dim3(a.n), dim3(256), 8 * p.splits * a.k, s, a, p.splits);
        return hipGetLastError();
    });
}

}  // namespace mg
