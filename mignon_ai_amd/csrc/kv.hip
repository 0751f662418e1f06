// A key/value cache in microscaled 4-bit blocks: rows quantised as they are written, read back, and attention over them with
// a sliding window and a few first positions (sinks) that stay visible.
#include "mx4.hpp"

#include <algorithm>

#include "common.hpp"
#include "mx4_device.hpp"

namespace mg {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// What a sequence's call covers: token t < count sits at position pos + t, the cache holds positions below `end`.
struct SeqSpan {
    int pos, count, end;
};
__device__ __forceinline__ SeqSpan seq_span(const int32_t* pos, const int32_t* counts, int s, int T) {
    SeqSpan r;
    r.pos = min(max(pos[s], -kKvMaxPos), kKvMaxPos);
    r.count = counts ? min(max(counts[s], 0), T) : T;
    r.end = r.pos + r.count;
    return r;
}
__device__ __forceinline__ int kv_slot(int p, int sinks, int ring) { return p < sinks ? p : sinks + (p - sinks) % ring; }

// ---- writing and reading rows --------------------------------------------------------------------------------------
// One launch for keys and values (blockIdx.z). DH / 8 lanes a row, four to a block; a workgroup covers 256 >> lc_log2 tokens
// by 1 << lc_log2 lanes of their heads * DH / 8.
template <int DH, class T, bool VEC>
__global__ __launch_bounds__(256) void kv_write_kernel(KvRowsArgs a, int lc_log2) {
    constexpr int LR = DH / 8;
    const int lanes = a.c.heads * LR, ring = a.c.cap - a.c.sinks, tokens = a.c.n * a.T;
    const int rows = 256 >> lc_log2, row_in = threadIdx.x >> lc_log2, c_in = threadIdx.x & ((1 << lc_log2) - 1);
    const KvRows& x = blockIdx.z ? a.v : a.k;
    uint8_t* codes = blockIdx.z ? a.c.v : a.c.k;
    uint8_t* scales = blockIdx.z ? a.c.vs : a.c.ks;
    for (long long m = (long long)blockIdx.x * rows + row_in; m < tokens; m += (long long)gridDim.x * rows) {
        const int s = (int)m / a.T, t = (int)m - s * a.T;
        const SeqSpan q = seq_span(a.pos, a.counts, s, a.T);
        const int p = q.pos + t;
        // a position that a later token of the same call takes the slot of is not written
        if (t >= q.count || p < 0 || (p >= a.c.sinks && p < q.end - ring)) continue;
        const int slot = kv_slot(p, a.c.sinks, ring);
        for (int c = (blockIdx.y << lc_log2) + c_in; c < lanes; c += gridDim.y << lc_log2) {
            const int h = c / LR, l = c - h * LR;
            float v[8];
            real_load8<T, VEC>((const T*)x.data + s * x.seq + t * x.token + h * x.head + 8 * l, 8, v);
            uint32_t sb;
            const uint32_t w = mx4_block(v, sb);
            const size_t row = ((size_t)s * a.c.heads + h) * a.c.cap + slot;
            *(uint32_t*)(codes + row * (DH / 2) + 4 * l) = w;
            if ((l & 3) == 0) scales[row * (DH / 32) + (l >> 2)] = (uint8_t)sb;
        }
    }
}

template <int DH, class T, bool VEC>
__global__ __launch_bounds__(256) void kv_read_kernel(KvRowsArgs a, int lc_log2) {
    constexpr int LR = DH / 8;
    const int lanes = a.c.heads * LR, ring = a.c.cap - a.c.sinks, tokens = a.c.n * a.T;
    const int rows = 256 >> lc_log2, row_in = threadIdx.x >> lc_log2, c_in = threadIdx.x & ((1 << lc_log2) - 1);
    const KvRows& x = blockIdx.z ? a.v : a.k;
    const uint8_t* codes = blockIdx.z ? a.c.v : a.c.k;
    const uint8_t* scales = blockIdx.z ? a.c.vs : a.c.ks;
    for (long long m = (long long)blockIdx.x * rows + row_in; m < tokens; m += (long long)gridDim.x * rows) {
        const int s = (int)m / a.T, t = (int)m - s * a.T;
        const SeqSpan q = seq_span(a.pos, a.counts, s, a.T);
        if (t >= q.count) continue;
        const int p = q.pos + t, end = a.lens ? min(max(a.lens[s], 0), kKvMaxPos) : q.end;
        const bool held = p >= 0 && p < end && (p < a.c.sinks || p >= end - ring);
        const int slot = held ? kv_slot(p, a.c.sinks, ring) : 0;
        for (int c = (blockIdx.y << lc_log2) + c_in; c < lanes; c += gridDim.y << lc_log2) {
            const int h = c / LR, l = c - h * LR;
            float v[8] = {};
            if (held) {
                const size_t row = ((size_t)s * a.c.heads + h) * a.c.cap + slot;
                mx4_unpack8(*(const uint32_t*)(codes + row * (DH / 2) + 4 * l), mx4_scale(scales[row * (DH / 32) + (l >> 2)]), v);
            }
            real_store8<T, VEC>((T*)x.data + s * x.seq + t * x.token + h * x.head + 8 * l, 8, v);
        }
    }
}

bool rows_aligned(const KvRows& r, int type) {
    const int e = real_size(type);
    return (uintptr_t)r.data % 16 == 0 && r.seq * e % 16 == 0 && r.token * e % 16 == 0 && r.head * e % 16 == 0;
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
    const int lanes = a.c.heads * a.c.dh / 8;
    int lc = 2;  // lanes is a multiple of 4
    while (lc < 8 && lanes % (2 << lc) == 0) lc++;
    const long long groups = ((long long)a.c.n * a.T + (256 >> lc) - 1) / (256 >> lc);
    const dim3 grid((unsigned)std::min<long long>(groups, 1 << 20), std::min(lanes >> lc, 32768), 2);
    const bool vec = rows_aligned(a.k, a.type) && rows_aligned(a.v, a.type);
    return by_width(a.c.dh, [&](auto w) {
        constexpr int DH = decltype(w)::value;
        return by_real(a.type, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if constexpr (READ) {
                if (vec) hipLaunchKernelGGL((kv_read_kernel<DH, T, true>), grid, dim3(256), 0, s, a, lc);
                else hipLaunchKernelGGL((kv_read_kernel<DH, T, false>), grid, dim3(256), 0, s, a, lc);
            } else {
                if (vec) hipLaunchKernelGGL((kv_write_kernel<DH, T, true>), grid, dim3(256), 0, s, a, lc);
                else hipLaunchKernelGGL((kv_write_kernel<DH, T, false>), grid, dim3(256), 0, s, a, lc);
            }
            return hipGetLastError();
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
    __device__ __forceinline__ int at(int o) const { return o < n0 ? o : o < n0 + n1 ? b1 + o - n0 : b2 + o - n0 - n1; }
};
// Rows at positions lo_row .. hi_row; the cache holds positions below `end`.
__device__ __forceinline__ Tiles tiles_of(int lo_row, int hi_row, int end, int sinks, int ring, int cap, int window) {
    Tiles r{0, 0, 0, 0, 0};
    if (hi_row < 0) return r;
    const int seen = min(sinks, hi_row + 1);
    r.n0 = (seen + 31) >> 5;
    int lo = max(sinks, end - ring);
    if (window > 0) lo = max(lo, lo_row - window + 1);
    if (hi_row < lo) return r;
    const int a = kv_slot(lo, sinks, ring) >> 5, b = (kv_slot(hi_row, sinks, ring) >> 5) + 1;
    const bool wraps = kv_slot(lo, sinks, ring) > kv_slot(hi_row, sinks, ring);
    r.b1 = max(r.n0, wraps ? sinks >> 5 : a);
    r.n1 = max(0, b - r.b1);
    if (wraps) {
        r.b2 = max(max(r.n0, r.b1 + r.n1), a);
        r.n2 = max(0, (cap >> 5) - r.b2);
    }
    return r;
}

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
//   Scores, K (16 keys a product) times q: step s of DH / 32 covers, for lane group g, channels (DH / 4) g + 8 s .. + 7, so
//   that a lane's steps are neighbouring words of a row (DH 96: channels 32 s + 8 g, since 24 do not end with a block).
//   Output, V^T times the probabilities: channels in chunks of 16 E, lane i owning E neighbouring ones (E 8, 4, 2).
template <int DH>
struct Width {
    static constexpr int KS = DH / 32;
    static constexpr bool kEven = DH != 96;
    static constexpr int chunks = DH == 96 ? 2 : 1;
    static constexpr int E0 = DH == 96 ? 4 : DH / 16;
    __device__ static constexpr int E(int c) { return c == 0 ? E0 : 2; }
    __device__ static int k_channel(int g, int s) { return kEven ? (DH / 4) * g + 8 * s : 32 * s + 8 * g; }
};

__device__ __forceinline__ float max_groups(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float sum_groups(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

constexpr int kTile = 32;
constexpr float kLog2e = 1.4426950408889634f;

// Few query rows: a wave takes 16 rows (the query heads of one key/value head, token after token) over a share of the tiles.
//
// Scores of 16 keys x 16 rows come out of the matrix cores with lane (i, g) holding row i and four keys; the keys of a tile
// are assigned to the product's rows so that group g ends with keys 8 g .. 8 g + 7, the very layout in which the second
// product takes the probabilities: they never leave their lane. V is brought into its layout (one channel of eight keys in
// a lane) by unpacking two keys' words and exchanging halves.
template <int DH, class T, int WAVES>
__global__ __launch_bounds__(256) void kv_attention_rows_kernel(KvAttnArgs a, int row_tiles, int chunk_tiles) {
    using W = Width<DH>;
    constexpr int QT = Terms<T>::q, PT = Terms<T>::p, ND = DH / 16, LD = DH + 4;
    __shared__ float s_ml[WAVES > 1 ? WAVES : 1][2][16];
    __shared__ float s_o[WAVES > 1 ? WAVES * 16 * LD : 1];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = WAVES > 1 ? blockIdx.x : blockIdx.x * 4 + wave, w = WAVES > 1 ? wave : 0;
    const int pairs = a.c.n * a.c.heads;
    if (unit >= pairs * row_tiles) return;
    const int pair = unit / row_tiles, rt = unit - pair * row_tiles;
    const int s = pair / a.c.heads, h = pair - s * a.c.heads;
    const SeqSpan q = seq_span(a.pos, a.counts, s, a.T);
    const int ring = a.c.cap - a.c.sinks, sinks = a.c.sinks;
    const int t_lo = rt * 16 / a.group;
    if (t_lo >= q.count) return;
    const int t_hi = min((rt * 16 + 15) / a.group, q.count - 1);
    const Tiles tl = tiles_of(q.pos + t_lo, q.pos + t_hi, q.end, sinks, ring, a.c.cap, a.window);
    const int n_tiles = tl.count();
    const int o0 = blockIdx.y * chunk_tiles, o1 = min(n_tiles, o0 + chunk_tiles);
    if (blockIdx.y && o0 >= n_tiles) return;

    // this lane's row
    const int row = rt * 16 + i, rows = a.T * a.group;
    const int t = row / a.group, head = h * a.group + (row - t * a.group);
    const bool there = row < rows && t < q.count;
    const int at = q.pos + t;
    v8bf qf[W::KS][QT];
#pragma unroll
    for (int st = 0; st < W::KS; st++) {
        float x[8] = {};
        if (there)
            real_load8<T, false>((const T*)a.q.data + s * a.q.seq + t * a.q.token + head * a.q.head + W::k_channel(g, st), 8, x);
        split_bf16<QT>(x, qf[st]);
    }
    const float scale = a.scale * kLog2e;

    // what the slots hold: slots of the ring up to `newest` belong to the run that ends with position end - 1
    const int last = q.end - 1, newest = last >= sinks ? kv_slot(last, sinks, ring) : -1;
    const size_t plane = (size_t)pair * a.c.cap;
    const uint8_t* kb = a.c.k + plane * (DH / 2);
    const uint8_t* ksb = a.c.ks + plane * (DH / 32);
    const uint8_t* vb = a.c.v + plane * (DH / 2);
    const uint8_t* vsb = a.c.vs + plane * (DH / 32);

    v4f acc[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) acc[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    uint32_t nan_blocks = 0;  // bit b: a key this row sees has NaN for channels 32 b .. 32 b + 31

    for (int o = o0 + w; o < o1; o += WAVES) {
        const int j0 = tl.at(o) * kTile;
        // scores
        float sc[8];
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const int key = j0 + (i >> 2) * 8 + 4 * hf + (i & 3);
            const uint8_t* kp = kb + (size_t)key * (DH / 2);
            const uint8_t* kss = ksb + (size_t)key * (DH / 32);
            v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int st = 0; st < W::KS; st++) {
                const int c0 = W::k_channel(g, st);
                const uint32_t word = *(const uint32_t*)(kp + c0 / 2);
                const float ks = mx4_scale(kss[c0 / 32]);
                uint32_t kw[4];
                kw[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, ks, 0));
                kw[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, ks, 1));
                kw[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, ks, 2));
                kw[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, ks, 3));
                const v8bf kf = __builtin_bit_cast(v8bf, *(uint4*)kw);
#pragma unroll
                for (int n = QT - 1; n >= 0; n--) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[st][n], d, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) sc[4 * hf + r] = d[r];
        }
        // who sees what: lane (i, g) holds row i and slots j0 + 8 g + e
        uint32_t sees = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int j = j0 + 8 * g + e;
            const int p = j < sinks ? j : last - (newest - j + (j > newest ? ring : 0));
            const bool held = j < sinks ? j <= last : p >= sinks;
            const bool v = held && p <= at && (j < sinks || a.window <= 0 || p > at - a.window);
            sees |= (uint32_t)v << e;
            sc[e] = v ? sc[e] * scale : -INFINITY;
        }
        float mt = sc[0];
#pragma unroll
        for (int e = 1; e < 8; e++) mt = fmaxf(mt, sc[e]);
        const float mn = fmaxf(m, max_groups(mt)), mu = mn == -INFINITY ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m - mu);
        m = mn;
        float p[8], ps = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = __builtin_amdgcn_exp2f(sc[e] - mu);
            ps += p[e];
        }
        l = l * al + ps;
#pragma unroll
        for (int d = 0; d < ND; d++) acc[d] *= al;
        v8bf pf[PT];
        split_bf16<PT>(p, pf);
        // output
#pragma unroll
        for (int c = 0; c < W::chunks; c++) {
            const int E = c == 0 ? W::E0 : 2, base = c == 0 ? 0 : 64, dt0 = c == 0 ? 0 : W::E0;
            const int blk = (base + i * E) / 32;
            uint32_t word[8], sb[8];
            uint32_t most = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const size_t key = (size_t)(j0 + 8 * g + e);
                const uint8_t* vp = vb + key * (DH / 2) + (base + i * E) / 2;
                word[e] = E == 8 ? *(const uint32_t*)vp : E == 4 ? *(const uint16_t*)vp : *vp;
                sb[e] = vsb[key * (DH / 32) + blk];
                most = max(most, sb[e]);
            }
            // a block of NaN stands apart: it would spread over rows that do not see its key (the writer's scales are at
            // most 252 otherwise; slots that were never written may hold anything)
            if (__any(most > 252u)) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const size_t key = (size_t)(j0 + 8 * g + e);
                    for (int b = 0; b < DH / 32; b++)
                        if (((sees >> e) & 1) && vsb[key * (DH / 32) + b] > 252u) nan_blocks |= 1u << b;
                    if (sb[e] > 252u) { sb[e] = 0; word[e] = 0; }
                }
            }
#pragma unroll
            for (int b = 0; b < E / 2; b++) {
                uint32_t lo[4], hi[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t x, y;
                    const float s0 = mx4_scale(sb[2 * e]), s1 = mx4_scale(sb[2 * e + 1]);
#define MX4_CVT(sel) \
    x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word[2 * e], s0, sel)); \
    y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word[2 * e + 1], s1, sel));
                    if (b == 0) { MX4_CVT(0) } else if (b == 1) { MX4_CVT(1) } else if (b == 2) { MX4_CVT(2) } else { MX4_CVT(3) }
#undef MX4_CVT
                    lo[e] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                    hi[e] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                }
                const v8bf v0 = __builtin_bit_cast(v8bf, *(uint4*)lo), v1 = __builtin_bit_cast(v8bf, *(uint4*)hi);
#pragma unroll
                for (int n = PT - 1; n >= 0; n--) {
                    acc[dt0 + 2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pf[n], acc[dt0 + 2 * b], 0, 0, 0);
                    acc[dt0 + 2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pf[n], acc[dt0 + 2 * b + 1], 0, 0, 0);
                }
            }
        }
    }
    l = sum_groups(l);
    nan_blocks |= __shfl_xor(nan_blocks, 16, 64);
    nan_blocks |= __shfl_xor(nan_blocks, 32, 64);
    if (nan_blocks) {
        // lane (i, g): row i, channels base + (4 g + r) E + e
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const bool first = d < W::E0;
            const int E = first ? W::E0 : 2, base = first ? 0 : 64, e = first ? d : d - W::E0;
#pragma unroll
            for (int r = 0; r < 4; r++)
                if ((nan_blocks >> ((base + (4 * g + r) * E + e) / 32)) & 1) acc[d][r] = NAN;
        }
    }
    const int chunks = (n_tiles + chunk_tiles - 1) / chunk_tiles;
    float total = l;
    if constexpr (WAVES > 1) {
        // join the waves: their sums at the largest maximum, added in the waves' order
        if (g == 0) {
            s_ml[w][0][i] = m;
            s_ml[w][1][i] = l;
        }
        __syncthreads();
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < WAVES; x++) top = fmaxf(top, s_ml[x][0][i]);
        const float tu = top == -INFINITY ? 0.0f : top;
        total = 0.0f;
#pragma unroll
        for (int x = 0; x < WAVES; x++) total += s_ml[x][1][i] * __builtin_amdgcn_exp2f(s_ml[x][0][i] - tu);
        const float f = __builtin_amdgcn_exp2f(m - tu);
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const bool first = d < W::E0;
            const int E = first ? W::E0 : 2, base = first ? 0 : 64, e = first ? d : d - W::E0;
#pragma unroll
            for (int r = 0; r < 4; r++) s_o[(w * 16 + i) * LD + base + (4 * g + r) * E + e] = acc[d][r] * f;
        }
        m = top;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const bool first = d < W::E0;
            const int E = first ? W::E0 : 2, base = first ? 0 : 64, e = first ? d : d - W::E0;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float v = 0.0f;
#pragma unroll
                for (int x = 0; x < WAVES; x++) v += s_o[(x * 16 + i) * LD + base + (4 * g + r) * E + e];
                acc[d][r] = v;
            }
        }
    }
    if (!there) return;
    float* part = nullptr;
    T* out = nullptr;
    float f = 1.0f;
    if (chunks > 1) {
        // [chunk][unit][row][DH + 2]: sums, maximum, sum of probabilities
        const int keep = min(16, rows);
        part = a.ws + (((size_t)blockIdx.y * pairs * row_tiles + unit) * keep + i) * (DH + 2);
        if (g == 0) {
            part[DH] = m;
            part[DH + 1] = total;
        }
    } else {
        out = (T*)a.out.data + s * a.out.seq + t * a.out.token + head * a.out.head;
        f = total == 0.0f ? 0.0f : 1.0f / total;
    }
#pragma unroll
    for (int d = 0; d < ND; d++) {
        const bool first = d < W::E0;
        const int E = first ? W::E0 : 2, base = first ? 0 : 64, e = first ? d : d - W::E0;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int ch = base + (4 * g + r) * E + e;
            if (part) part[ch] = acc[d][r];
            else out[ch] = (T)(acc[d][r] * f);
        }
    }
}

// Joins the chunks of a row tile that took more than one, in the chunks' order. A workgroup a row tile.
template <int DH, class T>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(KvAttnArgs a, int row_tiles, int chunk_tiles) {
    const int unit = blockIdx.x, pairs = a.c.n * a.c.heads;
    const int pair = unit / row_tiles, rt = unit - pair * row_tiles;
    const int s = pair / a.c.heads, h = pair - s * a.c.heads;
    const SeqSpan q = seq_span(a.pos, a.counts, s, a.T);
    const int t_lo = rt * 16 / a.group;
    if (t_lo >= q.count) return;
    const int t_hi = min((rt * 16 + 15) / a.group, q.count - 1);
    const Tiles tl = tiles_of(q.pos + t_lo, q.pos + t_hi, q.end, a.c.sinks, a.c.cap - a.c.sinks, a.c.cap, a.window);
    const int chunks = (tl.count() + chunk_tiles - 1) / chunk_tiles;
    if (chunks <= 1) return;
    const int rows = a.T * a.group, keep = min(16, rows);
    const size_t step = (size_t)pairs * row_tiles * keep * (DH + 2);
    for (int x = threadIdx.x; x < 16 * DH; x += 256) {
        const int i = x / DH, d = x - i * DH, row = rt * 16 + i;
        const int t = row / a.group, head = h * a.group + (row - t * a.group);
        if (row >= rows || t >= q.count) break;
        const float* part = a.ws + ((size_t)unit * keep + i) * (DH + 2);
        float top = -INFINITY;
        for (int c = 0; c < chunks; c++) top = fmaxf(top, part[c * step + DH]);
        const float tu = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, total = 0.0f;
        for (int c = 0; c < chunks; c++) {
            const float f = __builtin_amdgcn_exp2f(part[c * step + DH] - tu);
            sum += part[c * step + d] * f;
            total += part[c * step + DH + 1] * f;
        }
        T* out = (T*)a.out.data + s * a.out.seq + t * a.out.token + head * a.out.head;
        out[d] = (T)(total == 0.0f ? 0.0f : sum / total);
    }
}

struct RowsPlan {
    int row_tiles, units, waves, chunk_tiles, chunks;
};
RowsPlan rows_plan(const KvAttnArgs& a) {
    RowsPlan p;
    p.row_tiles = (a.T * a.group + 15) / 16;
    p.units = a.c.n * a.c.heads * p.row_tiles;
    // tiles a row tile can see, at most: the sinks', and the window's (or the ring's), with the ends of three runs
    const long long span = a.window > 0 ? std::min<long long>((long long)a.window + a.T, a.c.cap) : a.c.cap;
    const int tiles = (int)std::min<long long>((span + kTile - 1) / kTile + (a.c.sinks + kTile - 1) / kTile + 2, a.c.cap / kTile);
    p.waves = tiles <= 4 ? 1 : 4;
    p.chunk_tiles = tiles;
    if (p.waves > 1) {
        // enough workgroups to fill the chip, each with four tiles a wave at least
        const int want = std::max(1, 2048 / std::max(1, p.units));
        p.chunk_tiles = std::max(16, (tiles + want - 1) / want);
    }
    p.chunks = std::max(1, (tiles + p.chunk_tiles - 1) / p.chunk_tiles);
    return p;
}

}  // namespace

bool kv_head_width(int dh) { return dh == 32 || dh == 64 || dh == 96 || dh == 128; }

hipError_t launch_kv_write(const KvRowsArgs& a, hipStream_t s) { return launch_rows<false>(a, s); }
hipError_t launch_kv_read(const KvRowsArgs& a, hipStream_t s) { return launch_rows<true>(a, s); }

size_t kv_attention_ws_bytes(const KvAttnArgs& a) {
    const RowsPlan p = rows_plan(a);
    if (p.chunks <= 1) return 0;
    return (size_t)p.chunks * p.units * std::min(16, a.T * a.group) * (a.c.dh + 2) * 4;
}

hipError_t launch_kv_attention(const KvAttnArgs& a, hipStream_t s) {
    const RowsPlan p = rows_plan(a);
    return by_width(a.c.dh, [&](auto w) {
        constexpr int DH = decltype(w)::value;
        return by_real(a.type, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (p.waves == 1) {
                hipLaunchKernelGGL((kv_attention_rows_kernel<DH, T, 1>), dim3((p.units + 3) / 4), dim3(256), 0, s, a, p.row_tiles, p.chunk_tiles);
            } else {
                hipLaunchKernelGGL((kv_attention_rows_kernel<DH, T, 4>), dim3(p.units, p.chunks), dim3(256), 0, s, a, p.row_tiles, p.chunk_tiles);
                if (p.chunks > 1)
                    hipLaunchKernelGGL((kv_attention_join_kernel<DH, T>), dim3(p.units), dim3(256), 0, s, a, p.row_tiles, p.chunk_tiles);
            }
            return hipGetLastError();
        });
    });
}

}  // namespace mg
