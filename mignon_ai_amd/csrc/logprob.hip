// Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits.
//
// With m the largest logit of a row, S = sum e^(x - m) and X = sum (x - m) e^(x - m): log p(t) = (x_t - m) - log S, and the entropy is
// log S - X / S. One pass over the row: a lane keeps its own running maximum and sums, at 2^(x c - r) with c = log2 e and r = m c rounded,
// one fused operation a power; sums at one r are put at another by 2^(r - r'), and at the end r's rounding, d = m c - r, is taken out
// of log S (it cancels in the entropy).
//
// The k likeliest: of every 32 WAVES logits that lie in one of 64 groups of lanes, the largest; the k-th of these is at most the k-th of
// the tile, so only what reaches it can be among the k. Numbers and ids are one 64-bit key, no two alike: at most k groups, 32 k WAVES
// logits, reach the bound, whatever the logits are, and in ordinary rows few more than k. Later tiles are held to the bound so far, and
// one whose lanes' maxima all fail it (most do) costs nothing more. Candidates are put in order by counting, for each, those above it.
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

__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
template <int WAVES>
__device__ __forceinline__ void team_sync() {
    if constexpr (WAVES > 1) __syncthreads();
    else wave_fence();
}
template <int WAVES>
__device__ __forceinline__ bool team_any(bool v) {
    if constexpr (WAVES > 1) return __syncthreads_or(v);
    else return __any(v);
}

// The candidates of a team (a wave, or four) in LDS.
template <int WAVES>
struct Top {
    static constexpr int lanes = 64 * WAVES, each = 32 * WAVES;  // each: logits of a group in a tile
    uint64_t* keys;   // room
    uint64_t* best;   // 64 groups' keys; the k best in order
    int* count;
    int k, room, l;
    uint64_t bound = 1;
    static __host__ __device__ int room_of(int k) { return each * k + 256; }
    static __host__ __device__ int bytes(int k) { return k ? 8 * (room_of(k) + 64) + 16 : 0; }
    __device__ __forceinline__ Top(uint8_t* at, int k_, int l_) : k(k_), room(room_of(k_)), l(l_) {
        keys = (uint64_t*)at;
        best = keys + room;
        count = (int*)(best + 64);
    }
    // Raises the bound to the k-th largest of the groups' largest keys.
    __device__ void tighten(uint64_t mine) {
        if constexpr (WAVES > 1) {
            // four neighbouring lanes are a group
#pragma unroll
            for (int o = 1; o < WAVES; o *= 2) {
                const uint64_t other = __shfl_xor((unsigned long long)mine, o, 64);
                mine = other > mine ? other : mine;
            }
        }
        if (l % WAVES == 0) best[l / WAVES] = mine;
        team_sync<WAVES>();
        // (each wave finds it for itself)
        const uint64_t key = best[l & 63];
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < 64; j++) above += best[j] > key || (best[j] == key && j < (l & 63));  // (groups without logits are alike)
        const uint64_t who = __ballot(above == k - 1);
        const uint64_t kth = __shfl((unsigned long long)key, __ffsll((unsigned long long)who) - 1, 64);
        bound = kth > bound ? kth : bound;
        team_sync<WAVES>();
    }
    __device__ __forceinline__ void push(uint64_t key) {
        if (key < bound) return;
        const int at = atomicAdd(count, 1);
        if (at < room) keys[at] = key;
    }
    // Leaves the k largest of n candidates, in order, and raises the bound to the last of them.
    __device__ int select(int n) {
        for (int c = l; c < n; c += lanes) {
            const uint64_t key = keys[c];
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < n; j++) above += keys[j] > key;
            if (above < k) best[above] = key;
        }
        team_sync<WAVES>();
        const int left = min(n, k);
        if (l < left) keys[l] = best[l];
        if (l == 0) *count = left;
        if (left == k) bound = best[k - 1] > bound ? best[k - 1] : bound;
        team_sync<WAVES>();
        return left;
    }
};

// A team of WAVES waves takes a segment of a row, in tiles of 32 logits a lane, the next one loaded while one is worked on.
template <class T, int WAVES>
__global__ __launch_bounds__(256) void logprob_kernel(LogprobArgs a, int splits, int segment) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_part[3][4];
    constexpr int lanes = 64 * WAVES, tile = 32 * lanes, teams = 4 / WAVES;
    const int team = WAVES > 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & (lanes - 1);
    const long long unit = (long long)blockIdx.x * teams + team;
    if (unit >= (long long)a.n * splits) return;  // (a wave by itself)
    const long long r = splits == 1 ? unit : unit / splits;
    const int part = (int)(unit - r * splits), from = part * segment, to = min(a.V, from + segment);
    const T* x = (const T*)a.x + r * a.ld;
    Top<WAVES> top(smem + team * Top<WAVES>::bytes(a.k), a.k, l);

    Raw8<T> next[4];
    auto fetch = [&](int v0) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int v = v0 + (j * lanes + l) * 8;
            next[j].load(x + v, to - v);
        }
    };
    fetch(from);
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
        if (l == 0) *top.count = 0;
        team_sync<WAVES>();
    }
    for (int v0 = from; v0 < to; v0 += tile) {
        float y[32];
#pragma unroll
        for (int j = 0; j < 4; j++) next[j].get(y + 8 * j);
        if (v0 + tile < to) fetch(v0 + tile);
        float mt = y[0];
#pragma unroll
        for (int e = 1; e < 32; e++) mt = fmaxf(mt, y[e]);
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
        const bool first = v0 == from;
        if (!team_any<WAVES>(first || (top.bound >> 32) == 0 || mt >= key_value(top.bound))) continue;
        auto tighten = [&] {
            int id = -1;
            uint64_t key = 0;
#pragma unroll
            for (int e = 31; e >= 0; e--) {
                const int v = v0 + ((e >> 3) * lanes + l) * 8 + (e & 7);
                if (v < to) {
                    if (y[e] == mt) id = v;
                    else if (y[e] != y[e]) key = top_key(y[e], v);
                }
            }
            top.tighten(id >= 0 ? top_key(mt, id) : key);
        };
        auto push = [&] {
#pragma unroll
            for (int e = 0; e < 32; e++) {
                const int v = v0 + ((e >> 3) * lanes + l) * 8 + (e & 7);
                if (v < to) top.push(top_key(y[e], v));
            }
            team_sync<WAVES>();
        };
        if (first) tighten();
        push();
        int now = *top.count;
        if (now > top.room) {
            // more than there is room for reach the bound so far: once more, with the tile's own
            team_sync<WAVES>();
            if (l == 0) *top.count = n;
            team_sync<WAVES>();
            n = top.select(n);
            tighten();
            push();
            now = *top.count;
        }
        n = now;
        team_sync<WAVES>();
        if (n > 2 * a.k + 32) n = top.select(n);
    }
    // the row's: lanes' sums at the largest maximum
    float most = wave_max(m);
    if constexpr (WAVES > 1) {
        if ((l & 63) == 0) s_part[0][l >> 6] = most;
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
    if constexpr (WAVES > 1) {
        if ((l & 63) == 0) {
            s_part[1][l >> 6] = S;
            s_part[2][l >> 6] = X;
        }
        __syncthreads();
        S = (s_part[1][0] + s_part[1][1]) + (s_part[1][2] + s_part[1][3]);
        X = (s_part[2][0] + s_part[2][1]) + (s_part[2][2] + s_part[2][3]);
    }
    if (a.k) n = top.select(n);
    if (splits > 1) {
        uint8_t* out = (uint8_t*)a.ws + unit * part_bytes(a.k);
        if (most == -INFINITY) off = 0.0f;
        if (l == 0) {
            const float f = __builtin_amdgcn_exp2f(-off);
            *(Part*)out = Part{most, S * f, (X - off * S) * f, 0.0f};
        }
        uint64_t* keys = (uint64_t*)(out + sizeof(Part));
        if (l < a.k) keys[l] = l < n ? top.best[l] : 0;  // (k is at most 64)
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
        const uint64_t key = top.best[l];
        if (a.top_ids) a.top_ids[r * a.k + l] = key_id(key);
        if (a.top_logprob) a.top_logprob[r * a.k + l] = (key_value(key) - most) - log_s;
    }
}

// A row's segments: sums at the largest maximum, and the k largest of their k largest keys each. Of `splits` lists in order, the smallest of
// the ceil(k / splits)-th keys bounds the k-th of all.
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
    __shared__ uint64_t s_best[kMaxTop];
    __shared__ int s_count;
    if (l == 0) s_count = 0;
    const int deep = (a.k + splits - 1) / splits;
    uint64_t low = ~0ull;
    if (w < splits) low = ((const uint64_t*)(parts + w * part_bytes(a.k) + sizeof(Part)))[deep - 1];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)low, o, 64);
        low = other < low ? other : low;
    }
    __syncthreads();
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

struct LogprobPlan {
    int waves, splits, segment;
};
LogprobPlan logprob_plan(const LogprobArgs& a) {
    LogprobPlan p;
    p.waves = a.V <= 2048 ? 1 : 4;
    const int tile = 2048 * p.waves, tiles = (a.V - 1) / tile + 1;
    const int want = std::min(64, std::max(1, std::min(tiles, 1024 / std::max(a.n, 1))));
    p.segment = (tiles + want - 1) / want * tile;
    p.splits = (a.V - 1) / p.segment + 1;
    return p;
}

template <class T, int WAVES>
hipError_t launch_rows(const LogprobArgs& a, const LogprobPlan& p, hipStream_t s) {
    const long long units = (long long)a.n * p.splits;
    const int teams = 4 / WAVES;
    static std::atomic<uint64_t> allowed{0};
    if (const hipError_t e = allow_lds((const void*)logprob_kernel<T, WAVES>, teams * Top<WAVES>::bytes(kMaxTop), allowed); e != hipSuccess) return e;
    hipLaunchKernelGGL((logprob_kernel<T, WAVES>), dim3((unsigned)((units + teams - 1) / teams)), dim3(256), teams * Top<WAVES>::bytes(a.k), s, a,
                       p.splits, p.segment);
    return hipGetLastError();
}

}  // namespace

bool logprob_fits(const LogprobArgs& a) { return (long long)a.n * logprob_plan(a).splits < 1 << 24; }
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
