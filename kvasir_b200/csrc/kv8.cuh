// kv8.cuh -- the 8-bit KV cache: RoPE + quantising append, and reading rows back.
//
// A cache row (one position of one KV head) is head_dim 8-bit codes and one f32
// scale.  With amax = max |x| over the row and top = 127 (int8) or 448 (e4m3):
//   scale = amax / top,   code = round(x * (top / amax)),   value = code * scale.
// Both divisions are IEEE divisions and the product is one f32 multiply, so the
// codes are a function of the row alone.  |x * (top / amax)| <= top (1 + 2^-22),
// which rounds to at most top: nothing saturates.  A row whose amax is below
// 2^-119 (where top / amax would leave f32) is stored as zeros; a row with a NaN
// or an infinity gets a NaN scale and zero codes, so every element reads back NaN
// and attention over it gives NaN, as it does over a 16-bit cache.
//
// What is quantised is the row as the 16-bit cache holds it: K after the rotation's
// one rounding to 16 bits (rope.cuh's arithmetic), V as it is.
#pragma once

#include "rope.cuh"

namespace kvb {

constexpr float kKv8Tiny = 0x1p-119f;

template <int kFmt>
__host__ __device__ constexpr float kv8_top() {
    return kFmt == KVB_KV_INT8 ? 127.f : 448.f;
}

// Where the rows of a cache lie.  Contiguous: sequence b's rows start at b * seq_rows,
// [n_kv][max_seq].  Paged (block_table != nullptr): pools [n_blocks][n_kv][block_size];
// position p of sequence b lies in block block_table[b * max_blocks + p / block_size].
struct Kv8Place {
    uint8_t* kc;
    uint8_t* vc;
    float* ks;
    float* vs;
    long long seq_rows;
    int n_kv, hd, max_seq;
    const int32_t* block_table;
    int max_blocks, block_size, n_blocks;
};

// Row of (KV head 0, position p) of sequence b, and the rows between heads.  False (and
// reported) when the block entry lies outside the pool.
__device__ __forceinline__ bool kv8_row(const Kv8Place& a, int b, int p, size_t& row,
                                        size_t& head_rows, bool report) {
    if (!a.block_table) {
        row = (size_t)b * a.seq_rows + p;
        head_rows = (size_t)a.max_seq;
        return true;
    }
    const int lb = p / a.block_size;
    const int blk = a.block_table[(size_t)b * a.max_blocks + lb];
    if (blk < 0 || blk >= a.n_blocks) {
        if (report) raise_dev_error(kDevErrBadPosition);
        return false;
    }
    row = (size_t)blk * a.n_kv * a.block_size + (size_t)(p - lb * a.block_size);
    head_rows = (size_t)a.block_size;
    return true;
}

struct RowScale {
    float inv, scale;  // inv 0 with scale 0 or NaN: every code is 0
};
// From the largest magnitude's bit pattern: as unsigned integers the patterns order
// finite < inf < NaN, so a max over them never loses a NaN.
template <int kFmt>
__device__ __forceinline__ RowScale kv8_row_scale(uint32_t amax_bits) {
    RowScale r;
    const float amax = __uint_as_float(amax_bits);
    if (amax_bits >= 0x7f800000u) {
        r.inv = 0.f;
        r.scale = __uint_as_float(0x7fc00000u);
    } else if (amax < kKv8Tiny) {
        r.inv = 0.f;
        r.scale = 0.f;
    } else {
        r.inv = __fdiv_rn(kv8_top<kFmt>(), amax);
        r.scale = __fdiv_rn(amax, kv8_top<kFmt>());
    }
    return r;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Codes of two values in the low two bytes (a first).
template <int kFmt>
__device__ __forceinline__ uint32_t kv8_codes2(float a, float b, float inv) {
    if (inv == 0.f) return 0u;
    if (kFmt == KVB_KV_INT8) {
        return ((uint32_t)__float2int_rn(__fmul_rn(a, inv)) & 0xffu) |
               (((uint32_t)__float2int_rn(__fmul_rn(b, inv)) & 0xffu) << 8);
    } else {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
            : "=h"(r)
            : "f"(__fmul_rn(b, inv)), "f"(__fmul_rn(a, inv)));
        return r;
    }
}
// The value of one code (without its scale); exact.
template <int kFmt>
__device__ __forceinline__ float kv8_value(uint8_t c) {
    if (kFmt == KVB_KV_INT8) return (float)(int8_t)c;
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)c));
    const __half_raw h = {(unsigned short)(h2 & 0xffffu)};
    return __half2float(__half(h));
}

struct Kv8AppendArgs {
    uint16_t* qkv;
    int n_q, row_stride;
    int rows_per_seq;
    const int32_t* pos;
    const float* cos_t;  // nullptr: no rotation
    const float* sin_t;
    int max_pos;
    Kv8Place c;
};

// Any even head_dim <= 256, any alignment: one warp per (row, head), lane l holds the
// pairs l, l + 32, ... of the head's two halves.
template <typename T, int kFmt>
__global__ void __launch_bounds__(128) kv8_append_general_kernel(Kv8AppendArgs a, long long items) {
    const long long it = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (it >= items) return;
    const int heads = a.n_q + 2 * a.c.n_kv, hd = a.c.hd, half = hd >> 1;
    const int row = (int)(it / heads), h = (int)(it - (long long)row * heads);
    const int seq = row / a.rows_per_seq;
    const int p = a.pos[seq] + row % a.rows_per_seq;
    if (p < 0 || p >= a.c.max_seq || (a.cos_t && p >= a.max_pos)) {
        if (lane == 0) raise_dev_error(kDevErrBadPosition);
        return;
    }
    size_t crow, head_rows;
    if (!kv8_row(a.c, seq, p, crow, head_rows, lane == 0)) return;
    T* x = reinterpret_cast<T*>(a.qkv) + (size_t)row * a.row_stride + (size_t)h * hd;
    const bool rotate = a.cos_t && h < a.n_q + a.c.n_kv;
    float lo[4], hi[4];
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = lane + 32 * i;
        lo[i] = hi[i] = 0.f;
        if (j >= half) continue;
        lo[i] = Elem<T>::to_f(x[j]);
        hi[i] = Elem<T>::to_f(x[j + half]);
        if (rotate) {
            const float cs = a.cos_t[(size_t)p * half + j], sn = a.sin_t[(size_t)p * half + j];
            const T r0 = Elem<T>::from_f(rot_a(lo[i], hi[i], cs, sn));
            const T r1 = Elem<T>::from_f(rot_b(lo[i], hi[i], cs, sn));
            x[j] = r0;
            x[j + half] = r1;
            lo[i] = Elem<T>::to_f(r0);
            hi[i] = Elem<T>::to_f(r1);
        }
        mx = max(mx, max(abs_bits(lo[i]), abs_bits(hi[i])));
    }
    if (h < a.n_q) return;
    const RowScale rs = kv8_row_scale<kFmt>(__reduce_max_sync(0xffffffffu, mx));
    const bool is_v = h >= a.n_q + a.c.n_kv;
    crow += (size_t)(h - a.n_q - (is_v ? a.c.n_kv : 0)) * head_rows;
    uint8_t* dst = (is_v ? a.c.vc : a.c.kc) + crow * hd;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = lane + 32 * i;
        if (j >= half) continue;
        const uint32_t c2 = kv8_codes2<kFmt>(lo[i], hi[i], rs.inv);
        dst[j] = (uint8_t)c2;
        dst[j + half] = (uint8_t)(c2 >> 8);
    }
    if (lane == 0) (is_v ? a.c.vs : a.c.ks)[crow] = rs.scale;
}

struct Kv8ReadArgs {
    Kv8Place c;
    const int32_t* pos;
    int t, out_rows;  // rows read per sequence, rows per (sequence, head) of the outputs
    uint16_t* k_out;  // [n_seq][n_kv][out_rows][hd], rows 0 .. t-1 written
    uint16_t* v_out;
};

// Any head_dim, any alignment: one warp per (sequence, row, KV head, K or V).
template <typename T, int kFmt>
__global__ void __launch_bounds__(128) kv8_read_general_kernel(Kv8ReadArgs a, long long items) {
    const long long it = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (it >= items) return;
    const bool is_v = it & 1;
    const long long r = it >> 1;  // (sequence * n_kv + kv head) * t + i
    const int i = (int)(r % a.t);
    const long long bh = r / a.t;
    const int kvh = (int)(bh % a.c.n_kv), b = (int)(bh / a.c.n_kv);
    const int p = a.pos[b] + i;
    T* out = reinterpret_cast<T*>(is_v ? a.v_out : a.k_out) + ((size_t)bh * a.out_rows + i) * a.c.hd;
    size_t row = 0, head_rows = 0;
    bool ok = p >= 0 && p < a.c.max_seq;
    if (!ok && lane == 0) raise_dev_error(kDevErrBadPosition);
    ok = ok && kv8_row(a.c, b, p, row, head_rows, lane == 0);
    row += (size_t)kvh * head_rows;
    const float scale = ok ? (is_v ? a.c.vs : a.c.ks)[row] : 0.f;
    const uint8_t* src = (is_v ? a.c.vc : a.c.kc) + row * a.c.hd;
    for (int d = lane; d < a.c.hd; d += 32)
        out[d] = Elem<T>::from_f(ok ? kv8_value<kFmt>(src[d]) * scale : 0.f);
}

}  // namespace kvb
