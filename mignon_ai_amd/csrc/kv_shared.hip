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
// workgroup takes 32 rows a wave, RW waves, over a chunk of the prefix's tiles, which come into LDS as they are, three ahead, and are
// unpacked once for all waves while the tile before is worked on (the layouts are Unpacked's). All rows see all of a prefix, so there are
// no masks but behind its end, and a block of NaN belongs to every row.
template <int DH, class T, int RW>
__global__ __launch_bounds__(64 * RW, 2) void kv_prefix_kernel(KvSharedArgs a) {
    using W = Width<DH>;
    using Tile = KvTile<DH>;
    using U = Unpacked<DH>;
    constexpr int QT = Terms<T>::q, PT = Terms<T>::p, KF = DH / 16, ND = DH / 32, NT = 64 * RW, R = 32 * RW, o_raw = 2 * U::bytes;
    __shared__ __align__(16) uint8_t smem[o_raw + 3 * Tile::bytes];
    const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5, tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the row tile: of which prefix, and which of its tiles
    const int h = blockIdx.x % a.c.heads, per = a.T * a.group;  // rows a sequence
    int tile = blockIdx.x / a.c.heads, p = 0, first = 0;
    long long rows = 0;
    for (;; p++) {
        if (p == a.prefix.n) return;
        first = prefix_first(a, p);
        rows = (long long)max(prefix_first(a, p + 1) - first, 0) * per;
        const int tiles = (int)((rows + R - 1) / R);
        if (tile < tiles) break;
        tile -= tiles;
    }
    const PrefixSpan span = prefix_span(a, p);
    const int o0 = blockIdx.y * span.each, o1 = min(span.tiles, o0 + span.each);
    if (o0 >= o1) return;

    // this lane's row
    const long long row = (long long)tile * R + wave * 32 + i;
    const int s = first + (int)(min(row, rows - 1) / per), in = (int)(row - (long long)(s - first) * per);
    const int t = in / a.group, head = h * a.group + (in - t * a.group);
    const bool there = row < rows && t < (a.counts ? min(max(a.counts[s], 0), a.T) : a.T);
    if (!__syncthreads_or(there)) return;

    const size_t plane = ((size_t)p * a.c.heads + h) * a.prefix.cap;
    const uint32_t raw0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)(smem + o_raw);
    // loads of a tile: KS of 1 KiB, one of the scales, dealt out to the waves
    constexpr int loads = W::KS + 1, most = (loads + RW - 1) / RW;
    const int scales_from = min(4 * (W::NB == 3 ? lane : lane & (16 * W::NB - 1)), 64 * W::NB - 4);
    const uint8_t* scales = scales_from < 32 * W::NB ? a.prefix.ks + plane * W::NB + scales_from : a.prefix.vs + plane * W::NB + scales_from - 32 * W::NB;
    auto fetch = [&](int o, int slot) {
        const size_t j0 = (size_t)o * kTile;
#pragma unroll
        for (int x = 0; x < most; x++) {
            const int n = wave + RW * x;
            if (n < W::KS) {
                const int at = 1024 * n + 16 * lane;
                const uint8_t* from = at < Tile::half ? a.prefix.k + (plane + j0) * Tile::row + at : a.prefix.v + (plane + j0) * Tile::row + at - Tile::half;
                lds_load16(from, raw0 + slot * Tile::bytes + 1024 * n);
            } else if (n == W::KS) {
                lds_load4(scales + j0 * W::NB, raw0 + slot * Tile::bytes + Tile::o_scales);
            }
        }
    };
    const int mine = (loads - 1 - wave) / RW + (wave < loads ? 1 : 0);  // this wave's loads of a tile
    constexpr int words = DH / 8, NK = (32 * words + NT - 1) / NT, NV = (16 * words + NT - 1) / NT;
    int k_to[NK], v_from[NV], v_scale[NV], v_slot[NV], v_to[NV];
#pragma unroll
    for (int x = 0; x < NK; x++) {
        const int n = tid + NT * x, j = n / words, wd = n % words;
        k_to[x] = U::k_at(wd / 2, U::k_lane(j, wd & 1));
    }
#pragma unroll
    for (int x = 0; x < NV; x++) {
        const int n = tid + NT * x, j = n / words * 2, wd = n % words;
        v_from[x] = Tile::half + j * Tile::row + 4 * wd;
        v_scale[x] = Tile::o_scales + (32 + j) * W::NB + wd / 4;
        v_slot[x] = j;
        v_to[x] = U::v_at(wd / 4, j >> 4, U::v_lane(8 * (wd & 3), (j >> 2) & 1)) + 2 * ((j & 3) + (j >> 3 & 1) * 4);
    }
    auto unpack = [&](int raw, int buf, int j0) {
        const uint8_t* from = smem + o_raw + raw * Tile::bytes;
        uint8_t* out = smem + buf * U::bytes;
#pragma unroll
        for (int x = 0; x < NK; x++) {
            if (32 * words % NT && tid + NT * x >= 32 * words) break;
            const int n = tid + NT * x;  // (words and scales lie in the lanes' order)
            const uint32_t w = *(const uint32_t*)(from + 4 * n);
            const float sc = mx4_scale(from[Tile::o_scales + n / 4]);
            u32x4 y;
#pragma unroll
            for (int b = 0; b < 4; b++) y[b] = unpack2(w, sc, b);
            *(u32x4*)(out + k_to[x]) = y;
        }
#pragma unroll
        for (int x = 0; x < NV; x++) {
            if (16 * words % NT && tid + NT * x >= 16 * words) break;
            uint32_t w[2], sb[2];
#pragma unroll
            for (int y = 0; y < 2; y++) {
                w[y] = *(const uint32_t*)(from + v_from[x] + y * Tile::row);
                sb[y] = from[v_scale[x] + y * W::NB];
                if (j0 + v_slot[x] + y >= span.held) w[y] = sb[y] = 0;  // behind the end: may hold anything
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
    auto barrier = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    // the factor's sign, or zero, goes to the query, so that the largest product is the largest score
    const float sign = a.scale < 0.0f ? -1.0f : a.scale == 0.0f ? 0.0f : 1.0f, scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
    v8bf qf[KF][QT];
    {
        const T* q = (const T*)a.q.data + s * a.q.seq + t * a.q.token + head * a.q.head + 8 * g;
#pragma unroll
        for (int x = 0; x < KF; x++) {
            float y[8] = {};
            if (there) real_load8<T>(q + 16 * x, 8, y);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] *= sign;
            split_bf16<QT>(y, qf[x]);
        }
    }
    v16f acc[ND];
    float m, l;
    auto work = [&](auto careful, int buf, int j0) {
        const uint8_t* from = smem + buf * U::bytes;
        int k_lane = U::k_lane(i, g), v_lane = U::v_lane(i, g);
        asm volatile("" : "+v"(k_lane), "+v"(v_lane));
        v16f d = {};
#pragma unroll
        for (int x = 0; x < KF; x++) {
            const v8bf kf = *(const v8bf*)(from + U::k_at(x, k_lane));
#pragma unroll
            for (int n = QT - 1; n >= 0; n--) d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[x][n], d, 0, 0, 0);
        }
        if (j0 + 32 > span.held) {
            asm volatile("");
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (j0 + (r & 3) + 8 * (r >> 2) + 4 * g >= span.held) d[r] = -INFINITY;
        }
        float mt = d[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mt = fmaxf(mt, d[r]);
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
                const v8bf vf = *(const v8bf*)(from + U::v_at(x, hf, v_lane));
#pragma unroll
                for (int n = PT - 1; n >= 0; n--) acc[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[hf][n], acc[x], 0, 0, 0);
            }
    };
    auto sweep = [&](auto careful) {
#pragma unroll
        for (int x = 0; x < ND; x++) acc[x] = v16f{};
        m = -INFINITY;
        l = 0.0f;
        const int n = o1 - o0;
        for (int x = 0; x < min(n, 3); x++) fetch(o0 + x, x);
        vm_wait<0>();
        barrier();
        unpack(0, 0, o0 * kTile);
        int raw = 0;  // of tile x
        for (int x = 0; x < n; x++) {
            // tile x is unpacked, tile x + 1 has landed; tile x's raw place and the other unpacked one are free
            barrier();
            if (x + 3 < n) fetch(o0 + x + 3, raw);
            raw = raw == 2 ? 0 : raw + 1;
            if (x + 1 < n) unpack(raw, (x + 1) & 1, (o0 + x + 1) * kTile);
            work(careful, x & 1, (o0 + x) * kTile);
            // all but this step's loads have landed
            if (x + 3 >= n || mine == 0) vm_wait<0>();
            else if (mine == 1) vm_wait<1>();
            else vm_wait<most>();
        }
        barrier();
    };
    sweep(std::false_type());
    // scores far from zero: once more, with scores rounded as the maximum was (kFar)
    if (__syncthreads_or(m != -INFINITY && fabsf(m) >= kFar)) sweep(std::true_type());
    const float total = l + __shfl_xor(l, 32, 64);
    if (!there) return;
    // lane (i, g): row i, channels 32 x + 8 r + 4 g .. + 3
    const int heads = a.c.heads * a.group;
    float* part = a.parts + (((size_t)blockIdx.y * a.c.n + s) * a.T * heads + (size_t)t * heads + head) * kPart<DH>;
#pragma unroll
    for (int x = 0; x < ND; x++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            *(v4f*)(part + 32 * x + 8 * r + 4 * g) = v4f{acc[x][4 * r], acc[x][4 * r + 1], acc[x][4 * r + 2], acc[x][4 * r + 3]};
    if (g == 0) {
        part[DH] = m;
        part[DH + 1] = total;
    }
}

// How a call's rows are divided among workgroups of `rows` rows, and a prefix among `chunks`. How the sequences fall to the prefixes is
// not known here: there is room for a last, partly filled row tile each.
struct PrefixPlan {
    int rows, chunks;
    long long tiles;  // row tiles a head, at most
};
PrefixPlan prefix_plan(const KvSharedArgs& a) {
    PrefixPlan p;
    p.rows = 128;
    p.tiles = (long long)a.c.n * a.T * a.group / p.rows + a.prefix.n;
    const long long units = p.tiles * a.c.heads;
    p.chunks = (int)std::max<long long>(1, std::min<long long>(512 / units, a.prefix.cap / kTile / 8));
    return p;
}
size_t parts_bytes(const KvSharedArgs& a, const PrefixPlan& p) {
    return (size_t)p.chunks * a.c.n * a.T * a.c.heads * a.group * (a.c.dh + 4) * 4;
}

}  // namespace

// The parts, then the workspace of the rows' own attention.
size_t kv_shared_ws_bytes(const KvSharedArgs& a) {
    return own_ws_bytes(a, attn_plan(a)) + parts_bytes(a, prefix_plan(a));
}
bool kv_shared_fits(const KvSharedArgs& a) {
    return own_fits(attn_plan(a)) && prefix_plan(a).tiles * a.c.heads < 1 << 23;
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
            hipLaunchKernelGGL((kv_prefix_kernel<DH, T, 4>), dim3((unsigned)(p.tiles * a.c.heads), p.chunks), dim3(256), 0, s, a);
            return hipGetLastError();
        });
    });
    return e != hipSuccess ? e : launch_own_attention(a, s);
}

}  // namespace mg
