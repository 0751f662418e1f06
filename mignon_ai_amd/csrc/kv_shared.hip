// Attention for sequences that share prefixes: query rows over 4-bit prefixes, each read once for all of its sequences, and over every
// sequence's own 4-bit cache.
//
// A softmax over two sets of keys is the two sets' sums at their own maxima, put at the larger one: the first kernel gives each query
// row its prefix's largest score m, sum of powers l = sum 2^(score - m) and sum of values o, for every chunk of the prefix; the kernels
// of kv_attention.hpp then take the row's own positions and add those parts before they divide by the sum.
#include "kv_attention.hpp"

namespace mg {
namespace {

// ---- rows over a prefix --------------------------------------------------------------------------------------------
// The rows of a prefix and key/value head are those of all its sequences, tokens and the heads of the group, one after another. A
// workgroup takes 32 rows a wave, RW waves, over a chunk of the prefix, in steps of 64 slots. A step's codes are loaded straight to
// registers a step ahead, and unpacked once for all waves into one half of LDS while the waves work on the other (the layouts are
// Unpacked's); one barrier a step. All rows see all of a prefix, so there are no masks but behind its end, and a block of NaN belongs to
// every row.
//
// Bound by issuing: on this chip products and other vector instructions of a SIMD's waves take turns (8 products of 32 x 32 x 16 and 64
// fused multiply-adds a wave, four waves a SIMD: 1541 cycles, alone 1026 and 567), so a step costs a wave its 32 products, some 130
// other instructions and 32 powers, one after another, and its waits. Steps of 64 slots halve the waits of steps of 32: 32 x 32 tokens of 32
// query heads over 8 of 128, 16384 positions, bf16, 211 GFLOP: 334 -> 277 us (764 TFLOP/s; a large bf16 product reaches 1131); 64
// conversations 50 -> 35 (the checks of scales and scores below take 1 % of either). Not kept: a tile's scores among the powers of the one before (no gain), 64 rows a wave (registers moved to and
// fro, 503), three workgroups a CU (registers put to memory, 335), the scaled product of fp8 queries and the codes themselves (it drops
// what is 2^-13 of the largest product: errors of 1e-4 of the sum of magnitudes).
//
// For 16-bit queries values and probabilities are fp16, a probability as 2^15 times itself so that what is 2^-29 of a row's largest or less
// loses bits, not what is 2^-14: one product an output where two bf16 parts of a probability take two, at 11 bits instead of 16. fp16
// holds a 4-bit number exactly if its scale lies in 2^-23 .. 2^13 (bytes 104 to 140); a workgroup that meets another one (byte 0 with
// codes of zero is none: those are zeros), or scores far from zero (a maximum of kFar or more at any step: its rounding may put a
// probability past what fp16, or fp32, holds), goes over its tiles again in the careful form, which is that of kv_attention.hpp.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t unpack2h(uint32_t w, float s, int b) {
    switch (b) {
        case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0));
        case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1));
        case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2));
        default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3));
    }
}
template <bool HALF>
__device__ __forceinline__ uint32_t unpack2_as(uint32_t w, float s, int b) {
    return HALF ? unpack2h(w, s, b) : unpack2(w, s, b);
}
__device__ __forceinline__ v16f product(v8bf a, v8bf b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v16f product(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// What the two forms hold queries, keys, probabilities and values in, and in how many parts.
template <class T, bool CAREFUL>
struct Forms {
    static constexpr bool key_half = !CAREFUL && std::is_same_v<T, _Float16>, value_half = !CAREFUL && sizeof(T) == 2;
    using Q = std::conditional_t<key_half, v8h, v8bf>;
    using P = std::conditional_t<value_half, v8h, v8bf>;
    static constexpr int q = key_half ? 1 : Terms<T>::q, p = value_half ? 1 : Terms<T>::p;
    static constexpr float lift = value_half ? 15.0f : 0.0f;  // probabilities are held 2^lift times themselves
};
template <int N>
__device__ __forceinline__ void split(const float x[8], v8bf out[N]) { split_bf16<N>(x, out); }
template <int N>
__device__ __forceinline__ void split(const float x[8], v8h out[N]) {
    static_assert(N == 1, "");
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{x[2 * i], x[2 * i + 1]}), v2h));
    out[0] = __builtin_bit_cast(v8h, *(uint4*)w);
}

template <int DH, class T, int RW>
__global__ __launch_bounds__(64 * RW, sizeof(T) == 4 && DH >= 64 ? 1 : 2) void kv_prefix_kernel(KvSharedArgs a) {
    using W = Width<DH>;
    using U = Unpacked<DH>;
    constexpr int KF = DH / 16, ND = DH / 32, NT = 64 * RW, R = 32 * RW, row_bytes = DH / 2, step = 2 * U::bytes;
    __shared__ __align__(16) uint8_t smem[2 * step];
    const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5, tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the row tile: of which prefix, and which of its tiles (numbers without one, the last, come last); the chunk and the head
    const int h = blockIdx.x % a.c.heads, rest = blockIdx.x / a.c.heads, chunk = rest % a.prefix_chunks, per = a.T * a.group;  // rows a sequence
    int tile = rest / a.prefix_chunks, p = 0, first = 0;
    long long rows = 0;
    for (;; p += 64) {
        // 64 prefixes at once: their rows, their row tiles, and the tiles of those before
        if (p >= a.prefix.n) return;
        const int mine = p + lane, from = mine < a.prefix.n ? prefix_first(a, mine) : 0;
        const int count = mine < a.prefix.n ? max(prefix_first(a, mine + 1) - from, 0) : 0;
        const int tiles = (int)(((long long)count * per + R - 1) / R);
        int until = tiles;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int before = __shfl_up(until, o, 64);
            until += lane >= o ? before : 0;
        }
        const uint64_t past = __ballot(until > tile);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            tile -= __shfl(until - tiles, at, 64);
            first = __shfl(from, at, 64);
            rows = (long long)__shfl(count, at, 64) * per;
            p += at;
            break;
        }
        tile -= __shfl(until, 63, 64);
    }
    tile = __builtin_amdgcn_readfirstlane(tile);
    first = __builtin_amdgcn_readfirstlane(first);
    p = __builtin_amdgcn_readfirstlane(p);
    const PrefixSpan span = prefix_span(a, p);
    const int o0 = chunk * span.each, o1 = min(span.steps, o0 + span.each);
    if (o0 >= o1) return;

    // this lane's row
    const long long row = (long long)tile * R + wave * 32 + i;
    const int s = first + (int)(min(row, rows - 1) / per), in = (int)(row - (long long)(s - first) * per);
    const int t = in / a.group, head = h * a.group + (in - t * a.group);
    const bool there = row < rows && t < (a.counts ? min(max(a.counts[s], 0), a.T) : a.T);
    if (!__syncthreads_or(there)) return;

    // What a lane loads of a step, and where it unpacks it to: of K KV neighbouring words (of one block) of a slot, of V a word of each of two
    // neighbouring slots.
    constexpr int words = DH / 8, KW = 2 * kTile * words, VN = kTile * words;
    constexpr int KV = KW >= 4 * NT ? 4 : KW >= 2 * NT ? 2 : 1, KN = KW / KV, NK = (KN + NT - 1) / NT, NV = (VN + NT - 1) / NT;
    const size_t plane = ((size_t)p * a.c.heads + h) * a.prefix.cap;
    const uint8_t *kp = a.prefix.k + plane * row_bytes, *vp = a.prefix.v + plane * row_bytes, *ksp = a.prefix.ks + plane * W::NB, *vsp = a.prefix.vs + plane * W::NB;
    int k_to[NK][KV], v_to[NV];
#pragma unroll
    for (int x = 0; x < NK; x++)
#pragma unroll
        for (int e = 0; e < KV; e++) {
            const int n = (tid + NT * x) * KV + e, j = n / words, wd = n % words;
            k_to[x][e] = (j >> 5) * U::bytes + U::k_at(wd / 2, U::k_lane(j & 31, wd & 1));
        }
#pragma unroll
    for (int x = 0; x < NV; x++) {
        const int n = tid + NT * x, j = n / words * 2, wd = n % words;
        v_to[x] = (j >> 5) * U::bytes + U::v_at(wd / 4, (j >> 4) & 1, U::v_lane(8 * (wd & 3), (j >> 2) & 1)) + 2 * ((j & 3) + (j >> 3 & 1) * 4);
    }
    struct Raw {
        uint32_t k[NK][KV], ks[NK], v[NV][2], vs[NV][2];
    };
    // Slots behind the prefix's end may hold anything, or not be there: the last slot stands for them, its values with zeros.
    auto load = [&](Raw& w, int o) {
        const int j0 = o * 2 * kTile, last = span.held - 1 - j0;
        const uint8_t *k = kp + (size_t)j0 * row_bytes, *v = vp + (size_t)j0 * row_bytes, *ks = ksp + (size_t)j0 * W::NB, *vs = vsp + (size_t)j0 * W::NB;
#pragma unroll
        for (int x = 0; x < NK; x++) {
            if (KN % NT && tid + NT * x >= KN) break;
            const int n = (tid + NT * x) * KV, j = min(n / words, last), wd = n % words;
            if constexpr (KV == 4) *(u32x4*)w.k[x] = *(const u32x4*)(k + j * row_bytes + 4 * wd);
            else if constexpr (KV == 2) *(u32x2*)w.k[x] = *(const u32x2*)(k + j * row_bytes + 4 * wd);
            else w.k[x][0] = *(const uint32_t*)(k + j * row_bytes + 4 * wd);
            w.ks[x] = ks[j * W::NB + wd / 4];
        }
#pragma unroll
        for (int x = 0; x < NV; x++) {
            if (VN % NT && tid + NT * x >= VN) break;
            const int n = tid + NT * x, wd = n % words;
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int j = min(n / words * 2 + y, last);
                w.v[x][y] = *(const uint32_t*)(v + j * row_bytes + 4 * wd);
                w.vs[x][y] = vs[j * W::NB + wd / 4];
            }
        }
    };
    // Of scale bytes, and of them less 141, the least; byte 0 of a block of zeros (kSize: codes' bits without signs) counts as 104. low is 0
    // once a reference was far from zero, too.
    constexpr uint32_t kSize = 0x77777777u;
    uint32_t low = ~0u, high = ~0u;
    auto give = [&](auto careful, Raw& w, uint8_t* out, int o) {
        using Fm = Forms<T, decltype(careful)::value>;
        const int left = span.held - o * 2 * kTile;
#pragma unroll
        for (int x = 0; x < NK; x++) {
            if (KN % NT && tid + NT * x >= KN) break;
            if (Fm::key_half) {
                uint32_t least = w.ks[x];
                if (least == 0) {
                    asm volatile("");  // a branch: blocks of zeros are rare
                    uint32_t codes = 0;
#pragma unroll
                    for (int e = 0; e < KV; e++) codes |= w.k[x][e];
                    least = codes & kSize ? 0 : 104;
                }
                low = min(low, least);
                high = min(high, w.ks[x] - 141u);
            }
            const float sc = mx4_scale(w.ks[x]);
#pragma unroll
            for (int e = 0; e < KV; e++) {
                u32x4 y;
#pragma unroll
                for (int b = 0; b < 4; b++) y[b] = unpack2_as<Fm::key_half>(w.k[x][e], sc, b);
                *(u32x4*)(out + k_to[x][e]) = y;
            }
        }
        if (left < 2 * kTile) {
            asm volatile("");
#pragma unroll
            for (int x = 0; x < NV; x++)
#pragma unroll
                for (int y = 0; y < 2; y++)
                    if ((tid + NT * x) / words * 2 + y >= left) w.v[x][y] = w.vs[x][y] = 0;
        }
#pragma unroll
        for (int x = 0; x < NV; x++) {
            if (VN % NT && tid + NT * x >= VN) break;
            if (Fm::value_half) {
                uint32_t least = min(w.vs[x][0], w.vs[x][1]);
                if (least == 0) {
                    asm volatile("");
                    least = 104;
#pragma unroll
                    for (int y = 0; y < 2; y++) least = min(least, w.vs[x][y] == 0 && (w.v[x][y] & kSize) == 0 ? 104u : w.vs[x][y]);
                }
                low = min(low, least);
                high = min(high, min(w.vs[x][0] - 141u, w.vs[x][1] - 141u));
            }
            const float s0 = mx4_scale(w.vs[x][0]), s1 = mx4_scale(w.vs[x][1]);
#pragma unroll
            for (int b = 0; b < 4; b++) {
                // channels 8 wd + 2 b and the next
                const uint32_t y0 = unpack2_as<Fm::value_half>(w.v[x][0], s0, b), y1 = unpack2_as<Fm::value_half>(w.v[x][1], s1, b);
                *(uint32_t*)(out + (v_to[x] ^ (32 * b))) = __builtin_amdgcn_perm(y1, y0, 0x05040100u);
                *(uint32_t*)(out + (v_to[x] ^ (32 * b + 16))) = __builtin_amdgcn_perm(y1, y0, 0x07060302u);
            }
        }
    };
    auto barrier = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    // the factor's sign, or zero, goes to the query, so that the largest product is the largest score
    const float sign = a.scale < 0.0f ? -1.0f : a.scale == 0.0f ? 0.0f : 1.0f, scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
    v16f acc[ND];
    float ref, l;  // 2^-ref is in l and acc
    auto sweep = [&](auto careful) {
        constexpr bool CAREFUL = decltype(careful)::value;
        using Fm = Forms<T, CAREFUL>;
        typename Fm::Q qf[KF][Fm::q];
        const T* q = (const T*)a.q.data + s * a.q.seq + t * a.q.token + head * a.q.head + 8 * g;
#pragma unroll
        for (int x = 0; x < KF; x++) {
            float y[8] = {};
            if (there) real_load8<T>(q + 16 * x, 8, y);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] *= sign;
            split<Fm::q>(y, qf[x]);
        }
#pragma unroll
        for (int x = 0; x < ND; x++) acc[x] = v16f{};
        float m = -INFINITY;  // the largest product so far
        ref = -Fm::lift;
        l = 0.0f;
        Raw w;
        // Step o, unpacked in half `buf`; the next one is unpacked meanwhile, and the one after that asked for.
        auto work = [&](auto buf, int o) {
            uint8_t* from = smem + decltype(buf)::value * step;
            uint8_t* to = smem + (1 - decltype(buf)::value) * step;
            // All fragments of a product are asked for before the first is needed, V's before the softmax: left to itself the compiler waits for
            // them two by two.
            constexpr bool EARLY = !CAREFUL && sizeof(T) == 2;
            constexpr int AHEAD = DH <= 64 ? 2 : 1;
            const auto key = [&](int u, int f) { return *(const typename Fm::Q*)(from + u * U::bytes + U::k_at(f, U::k_lane(i, g))); };
            const auto value = [&](int u, int f) { return *(const typename Fm::P*)(from + u * U::bytes + U::v_at(f >> 1, f & 1, U::v_lane(i, g))); };
            typename Fm::Q kf[2][KF];
            typename Fm::P vf[2][2 * ND];
            if (EARLY) {
#pragma unroll
                for (int f = 0; f < KF; f++)
#pragma unroll
                    for (int u = 0; u < 2; u++) kf[u][f] = key(u, f);
                __builtin_amdgcn_sched_barrier(0);
            }
            v16f d[2] = {v16f{}, v16f{}};
#pragma unroll
            for (int f = 0; f < KF; f++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (!EARLY) kf[u][f] = key(u, f);
#pragma unroll
                    for (int n = Fm::q - 1; n >= 0; n--) d[u] = product(kf[u][f], qf[f][n], d[u]);
                }
            if (EARLY) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int f = 0; f < 2 * ND; f++)
#pragma unroll
                    for (int u = 0; u < AHEAD; u++) vf[u][f] = value(u, f);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (o + 1 < o1) give(careful, w, to, o + 1);
            if (o + 2 < o1) load(w, o + 2);
            const int left = span.held - o * 2 * kTile;
            if (left < 2 * kTile) {
                asm volatile("");
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (kTile * u + (r & 3) + 8 * (r >> 2) + 4 * g >= left) d[u][r] = -INFINITY;
            }
            float mt = d[0][0];
#pragma unroll
            for (int r = 1; r < 32; r++) mt = __builtin_elementwise_maximum(mt, d[r >> 4][r & 15]);
            if (__any(mt > m)) {  // rare after the first steps
                const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
                const float mn = fmaxf(m, fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])));
                const float now = mn == -INFINITY ? -Fm::lift : mn * scale - Fm::lift;
                const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ref - now);  // (0: there is nothing yet)
                if (fabsf(now) >= kFar) low = 0;  // (also where a nearer one follows)
                m = mn;
                ref = now;
                l *= al;
#pragma unroll
                for (int f = 0; f < ND; f++) acc[f] *= al;
            }
            typename Fm::P pf[2][2][Fm::p];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                float pr[16];
#pragma unroll
                for (int r = 0; r < 16; r++)
                    pr[r] = __builtin_amdgcn_exp2f(CAREFUL && fabsf(ref) >= kFar ? d[u][r] * scale - ref : fmaf(d[u][r], scale, -ref));
                split<Fm::p>(pr, pf[u][0]);
                split<Fm::p>(pr + 8, pf[u][1]);
                if constexpr (Fm::value_half) {
                    // (the probabilities as they are held)
                    const v2h one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int e = 0; e < 4; e++) l = __builtin_amdgcn_fdot2(v2h{pf[u][hf][0][2 * e], pf[u][hf][0][2 * e + 1]}, one, l, false);
                } else {
                    float sum[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) sum[r] = (pr[r] + pr[4 + r]) + (pr[8 + r] + pr[12 + r]);
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                }
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int f = 0; f < 2 * ND; f++) {
                    if (!EARLY || u >= AHEAD) vf[u][f] = value(u, f);
#pragma unroll
                    for (int n = Fm::p - 1; n >= 0; n--) acc[f >> 1] = product(vf[u][f], pf[u][f & 1][n], acc[f >> 1]);
                }
        };
        load(w, o0);
        give(careful, w, smem, o0);
        if (o0 + 1 < o1) load(w, o0 + 1);
        for (int o = o0; o < o1; o += 2) {
            barrier();
            work(std::integral_constant<int, 0>(), o);
            if (o + 1 < o1) {
                barrier();
                work(std::integral_constant<int, 1>(), o + 1);
            }
        }
        barrier();
    };
    sweep(std::false_type());
    if (__syncthreads_or(low < 104u || high < 114u)) sweep(std::true_type());
    const float total = l + __shfl_xor(l, 32, 64);
    if (!there) return;
    // lane (i, g): row i, channels 32 x + 8 r + 4 g .. + 3
    const int heads = a.c.heads * a.group;
    float* part = a.parts + (((size_t)chunk * a.c.n + s) * a.T * heads + (size_t)t * heads + head) * kPart<DH>;
#pragma unroll
    for (int x = 0; x < ND; x++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            *(v4f*)(part + 32 * x + 8 * r + 4 * g) = v4f{acc[x][4 * r], acc[x][4 * r + 1], acc[x][4 * r + 2], acc[x][4 * r + 3]};
    if (g == 0) {
        part[DH] = total == 0.0f ? -INFINITY : ref;
        part[DH + 1] = total;
    }
}

// How a call's rows are divided among workgroups of `rows` rows, and a prefix among `chunks`. How the sequences fall to the prefixes, and
// how long these are, is not known here: there is room for a last, partly filled row tile each.
//
// Eight waves share a workgroup's unpacking where heads are wide, rows are 16-bit and a prefix has 256 or more of a head, four elsewhere (us
// of this kernel, four and eight waves at their best chunks, bf16 heads of 128: 1024 rows of each of 8 heads over 16384 positions, four
// times, 304 and 277; 256 rows over 16384 40 and 35; fp16 heads of 64, 680 rows over up to 6001, 22 and 26). Workgroups for every CU, of four
// waves three, each with two steps at least; more cost more at their ends and in the join (the 256 rows with 8, 16 and 32 chunks 76, 48 and 35,
// with 64 each 2 steps less; the 680 rows with 4, 8, 16 chunks 30, 21.7, 22.9; 8 fp32 heads of 32, 820 rows over up to 1000, with 1, 2, 3, 4:
// 28, 20.6, 17.8, 27.3).
struct PrefixPlan {
    int rows, chunks;
    long long tiles;  // row tiles a head, at most
};
PrefixPlan prefix_plan(const KvSharedArgs& a) {
    PrefixPlan p;
    const long long all = (long long)a.c.n * a.T * a.group;  // of a head
    p.rows = real_size(a.type) == 2 && a.c.dh >= 96 && all >= 256LL * a.prefix.n ? 256 : 128;
    p.tiles = std::max(0LL, all - a.prefix.n) / p.rows + a.prefix.n;
    const long long want = (p.rows == 256 ? 256 : 768) / std::max(1LL, p.tiles * a.c.heads);
    p.chunks = (int)std::max<long long>(1, std::min<long long>(want, a.prefix.cap / (2 * kTile) / 2));
    return p;
}
size_t parts_bytes(const KvSharedArgs& a, const PrefixPlan& p) {
    return (size_t)p.chunks * a.c.n * a.T * a.c.heads * a.group * (a.c.dh + 4) * 4;
}

}  // namespace

// The parts, then the workspace of the rows' own attention; for rows of any type.
size_t kv_shared_ws_bytes(const KvSharedArgs& a) {
    size_t parts = 0;
    for (const int type : {REAL_F32, REAL_BF16}) {
        KvSharedArgs b = a;
        b.type = type;
        parts = std::max(parts, parts_bytes(b, prefix_plan(b)));
    }
    return own_ws_bytes(a, attn_plan(a)) + parts;
}
bool kv_shared_fits(const KvSharedArgs& a) {
    const PrefixPlan p = prefix_plan(a);
    return own_fits(attn_plan(a)) && p.tiles * a.c.heads * p.chunks < 1 << 23;
}

hipError_t launch_kv_shared(const KvSharedArgs& args, hipStream_t s) {
    KvSharedArgs a = args;
    const PrefixPlan p = prefix_plan(a);
    a.prefix_chunks = p.chunks;
    a.parts = a.ws;
    a.ws = (float*)((char*)a.ws + parts_bytes(a, p));
    const hipError_t e = by_width(a.c.dh, [&](auto w) {
        constexpr int DH = decltype(w)::value;
        return by_real(a.type, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            const dim3 grid((unsigned)(p.tiles * p.chunks * a.c.heads));
            if constexpr (sizeof(T) == 2 && DH >= 96) {
                if (p.rows == 256) {
                    hipLaunchKernelGGL((kv_prefix_kernel<DH, T, 8>), grid, dim3(512), 0, s, a);
                    return hipGetLastError();
                }
            }
            hipLaunchKernelGGL((kv_prefix_kernel<DH, T, 4>), grid, dim3(256), 0, s, a);
            return hipGetLastError();
        });
    });
    return e != hipSuccess ? e : launch_own_attention(a, s);
}

}  // namespace mg
