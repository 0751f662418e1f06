// The microscaled 4-bit format (blocks of 32 elements in E2M1 with one power-of-two scale byte, E8M0): quantisation,
// product, and a key/value cache held in it (see mx4.hip, kv.hip; no reference counterpart).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mg {

// Element types of real-valued arrays (MG_F32, MG_F16, MG_BF16).
enum RealType : int { REAL_F32 = 0, REAL_F16 = 1, REAL_BF16 = 2 };
constexpr int real_size(int type) { return type == REAL_F32 ? 4 : 2; }

// Operand rows are padded to whole 128-element steps: Kp = round_up(K, 128), Kp / 2 code bytes and Kp / 32 scale bytes a row.
struct Mx4RowsArgs {
    const void* x = nullptr;   // quantise: rows [M][K], row stride ldx elements
    void* y = nullptr;         // dequantise: the same
    int type = REAL_F32;
    int M = 0, K = 0;
    long long ld = 0;
    uint8_t* codes = nullptr;
    uint8_t* scales = nullptr;
};
hipError_t launch_mx4_quantize(const Mx4RowsArgs& a, hipStream_t s);
hipError_t launch_mx4_dequantize(const Mx4RowsArgs& a, hipStream_t s);

struct Mx4GemmArgs {
    const uint8_t* A = nullptr;   // codes [M][Kp / 2], scales [M][Kp / 32]
    const uint8_t* As = nullptr;
    const uint8_t* W = nullptr;   // codes [N][Kp / 2], scales [N][Kp / 32]
    const uint8_t* Ws = nullptr;
    int M = 0, N = 0, Kp = 0;
    void* C = nullptr;            // [M][N]
    int type = REAL_F32;
};
bool mx4_gemm_fits(const Mx4GemmArgs& a);  // a launch takes it
hipError_t launch_mx4_gemm(const Mx4GemmArgs& a, hipStream_t s);

// Rows of a cache call: element (sequence s, token t, head h, channel d) at data + s * seq + t * token + h * head + d.
struct KvRows {
    void* data = nullptr;
    long long seq = 0, token = 0, head = 0;
};
// A cache of n sequences: position p < sinks in slot p, a later one in slot sinks + (p - sinks) % (cap - sinks).
struct KvCache {
    int n = 0, heads = 0, dh = 0, cap = 0, sinks = 0;
    uint8_t* k = nullptr;         // codes [n][heads][cap][dh / 2]
    uint8_t* ks = nullptr;        // scales [n][heads][cap][dh / 32]
    uint8_t* v = nullptr;
    uint8_t* vs = nullptr;
};
// Token t < counts[s] (null: T) of sequence s sits at position pos[s] (null: 0) + t.
struct KvRowsArgs {
    KvCache c;
    KvRows k, v;
    int type = REAL_F32, T = 0;
    const int32_t* pos = nullptr;
    const int32_t* counts = nullptr;
    const int32_t* lens = nullptr;  // read: the sequences' lengths, null: pos + counts
};
hipError_t launch_kv_write(const KvRowsArgs& a, hipStream_t s);
hipError_t launch_kv_read(const KvRowsArgs& a, hipStream_t s);

struct KvAttnArgs {
    KvCache c;
    KvRows q, out;                // heads * group query heads; query head i reads key/value head i / group
    int type = REAL_F32, T = 0, group = 1, window = 0;
    float scale = 1.0f;
    const int32_t* pos = nullptr;
    const int32_t* counts = nullptr;
    float* ws = nullptr;          // kv_attention_ws_bytes
};
// Positions are below this.
constexpr int kKvMaxPos = 1 << 30;
bool kv_head_width(int dh);       // 32, 64, 96 or 128
size_t kv_attention_ws_bytes(const KvAttnArgs& a);
bool kv_attention_fits(const KvAttnArgs& a);  // a launch takes it
hipError_t launch_kv_attention(const KvAttnArgs& a, hipStream_t s);

}  // namespace mg
