// A key/value cache in microscaled 4-bit blocks: rows quantised as they are written, read back, and attention over them with
// a sliding window and a few first positions (sinks) that stay visible.
#include "kv_attention.hpp"

namespace mg {
namespace {

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

}  // namespace

bool kv_head_width(int dh) { return dh == 32 || dh == 64 || dh == 96 || dh == 128; }

hipError_t launch_kv_write(const KvRowsArgs& a, hipStream_t s) { return launch_rows<false>(a, s); }
hipError_t launch_kv_read(const KvRowsArgs& a, hipStream_t s) { return launch_rows<true>(a, s); }

size_t kv_attention_ws_bytes(const KvAttnArgs& a) { return own_ws_bytes(a, attn_plan(a)); }
bool kv_attention_fits(const KvAttnArgs& a) { return own_fits(attn_plan(a)); }
hipError_t launch_kv_attention(const KvAttnArgs& a, hipStream_t s) { return launch_own_attention(a, s); }

}  // namespace mg
