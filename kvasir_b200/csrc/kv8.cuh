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

// The values of four codes, in order; exact.  int8: 2^23 + 128 + code is the f32 whose low
// byte is the code plus 128.
template <int kFmt>
__device__ __forceinline__ void kv8_values4(uint32_t w, float* x) {
    if (kFmt == KVB_KV_INT8) {
        const uint32_t u = w ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t v;
            asm("prmt.b32 %0, %1, %2, %3;" : "=r"(v) : "r"(u), "r"(0x4b000000u), "r"(0x7440u | i));
            x[i] = __uint_as_float(v) - 8388736.f;
        }
    } else {
        uint32_t lo, hi;
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
        const float2 a = Elem<__half>::unpack(lo), b = Elem<__half>::unpack(hi);
        x[0] = a.x;
        x[1] = a.y;
        x[2] = b.x;
        x[3] = b.y;
    }
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

// Eight codes of values x (already 16-bit values in f32), packed in order.
// int8: x * inv plus 1.5 * 2^23 leaves the integer rounded to nearest even in the low bits
// of the sum; the multiply and the add are kept apart, as the definition rounds the product.
template <int kFmt>
__device__ __forceinline__ uint2 kv8_codes8(const float* x, float inv) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (kFmt == KVB_KV_INT8) {
            uint32_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v[k] = __float_as_uint(__fadd_rn(__fmul_rn(x[4 * i + k], inv), 12582912.f));
            uint32_t lo, hi;
            asm("prmt.b32 %0, %1, %2, 0x0040;" : "=r"(lo) : "r"(v[0]), "r"(v[1]));
            asm("prmt.b32 %0, %1, %2, 0x0040;" : "=r"(hi) : "r"(v[2]), "r"(v[3]));
            asm("prmt.b32 %0, %1, %2, 0x5410;" : "=r"(w[i]) : "r"(lo), "r"(hi));
        } else {
            w[i] = kv8_codes2<kFmt>(x[4 * i], x[4 * i + 1], inv) |
                   (kv8_codes2<kFmt>(x[4 * i + 2], x[4 * i + 3], inv) << 16);
        }
    }
    return inv == 0.f ? make_uint2(0u, 0u) : make_uint2(w[0], w[1]);
}

// Magnitudes of two packed 16-bit elements against the running maxima: as unsigned integers
// the patterns order finite < inf < NaN in both types.
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t v) {
    return __vmaxu2(m, v & 0x7fff7fffu);
}
// The f32 bit pattern of a 16-bit magnitude's pattern (order kept: NaN > inf > finite).
template <typename T>
__device__ __forceinline__ uint32_t widen_bits(uint32_t h) {
    return __float_as_uint(Elem<T>::unpack(h).x) & 0x7fffffffu;
}

// head_dim = 16 CPR (64 or 128), 16-byte aligned rows and tables: one CTA per qkv row, a
// thread per chunk of 8 pairs (elements 8j .. and 8j + head_dim / 2 ..) of a head, so that
// the CPR threads of a head are neighbours and its largest magnitude takes log2 CPR
// shuffles.  Both 16-byte loads of a thread are issued before its position is known, the
// rotation goes four pairs at a time and the maximum over packed elements: 40 registers,
// so that 1,536 threads (48 KB of loads) are in flight on an SM -- at 62 registers 960 were,
// and 4 x 2048 tokens of 32 + 16 heads (103 MB) took 25 us instead of 21.2 (with 24 bytes a thread
// spilled).  Measured no
// better: 48 registers with several short rows per CTA (21.2), a persistent grid that requests
// the next row ahead (28.3).  What bounds it is issue (61 % of slots, 75 % of an SM's busy
// time).  Packed f32x2 multiplies and adds would halve the arithmetic, but the assembler
// contracts them into one rounding (x * inv = 63.5 - 2^-18 then gives code 63, not 64).
template <typename T, int kFmt, int CPR>
__global__ void __launch_bounds__(256, 6) kv8_append_vec_kernel(Kv8AppendArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int hd = 16 * CPR, half = 8 * CPR;
    const int row = blockIdx.x;
    const int seq = row / a.rows_per_seq;
    const int heads = a.n_q + 2 * a.c.n_kv, items = heads * CPR;
    const int n_rot = a.n_q + a.c.n_kv;
    uint16_t* rowp = a.qkv + (size_t)row * a.row_stride;
    bool placed = false;
    size_t crow0 = 0, head_rows = 0;
    // whole warps take part (shuffles); threads past the last item only keep them company
    for (int it0 = threadIdx.x & ~31; it0 < items; it0 += blockDim.x) {
        const int it = it0 + (threadIdx.x & 31);
        const bool have = it < items;
        const int h = it / CPR, j = it % CPR;
        uint4* pa = reinterpret_cast<uint4*>(rowp + h * hd + 8 * j);
        uint4* pb = reinterpret_cast<uint4*>(rowp + h * hd + 8 * j + half);
        uint4 va = make_uint4(0u, 0u, 0u, 0u), vb = va;
        if (have) {
            va = *pa;
            vb = *pb;
        }
        const int p = a.pos[seq] + (row - seq * a.rows_per_seq);
        if (!placed) {
            placed = true;
            if (p < 0 || p >= a.c.max_seq || (a.cos_t && p >= a.max_pos)) {
                if (threadIdx.x == 0) raise_dev_error(kDevErrBadPosition);
                return;
            }
            if (!kv8_row(a.c, seq, p, crow0, head_rows, threadIdx.x == 0)) return;
        }
        if (have && a.cos_t && h < n_rot) {
            const float4* c4 = reinterpret_cast<const float4*>(a.cos_t + (size_t)p * half + 8 * j);
            const float4* s4 = reinterpret_cast<const float4*>(a.sin_t + (size_t)p * half + 8 * j);
            auto rotate2 = [](uint32_t& lo, uint32_t& hi, float c0, float c1, float s0, float s1) {
                const float2 x = Elem<T>::unpack(lo), y = Elem<T>::unpack(hi);
                lo = Elem<T>::pack(rot_a(x.x, y.x, c0, s0), rot_a(x.y, y.y, c1, s1));
                hi = Elem<T>::pack(rot_b(x.x, y.x, c0, s0), rot_b(x.y, y.y, c1, s1));
            };
            float4 c = c4[0], sn = s4[0];
            rotate2(va.x, vb.x, c.x, c.y, sn.x, sn.y);
            rotate2(va.y, vb.y, c.z, c.w, sn.z, sn.w);
            c = c4[1];
            sn = s4[1];
            rotate2(va.z, vb.z, c.x, c.y, sn.x, sn.y);
            rotate2(va.w, vb.w, c.z, c.w, sn.z, sn.w);
            *pa = va;
            *pb = vb;
        }
        if (it0 + 31 < a.n_q * CPR) continue;  // a warp of query heads
        uint32_t m2 = max_abs2(max_abs2(max_abs2(max_abs2(0u, va.x), va.y), va.z), va.w);
        m2 = max_abs2(max_abs2(max_abs2(max_abs2(m2, vb.x), vb.y), vb.z), vb.w);
        uint32_t mx = max(m2 & 0xffffu, m2 >> 16);
#pragma unroll
        for (int o = 1; o < CPR; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (!have || h < a.n_q) continue;
        const RowScale rs = kv8_row_scale<kFmt>(widen_bits<T>(mx));
        const bool is_v = h >= n_rot;
        const size_t crow = crow0 + (size_t)(h - (is_v ? n_rot : a.n_q)) * head_rows;
        uint8_t* dst = (is_v ? a.c.vc : a.c.kc) + crow * hd + 8 * j;
        float x[8];
        unpack8<T>(va, x);
        *reinterpret_cast<uint2*>(dst) = kv8_codes8<kFmt>(x, rs.inv);
        unpack8<T>(vb, x);
        *reinterpret_cast<uint2*>(dst + half) = kv8_codes8<kFmt>(x, rs.inv);
        if (j == 0) (is_v ? a.c.vs : a.c.ks)[crow] = rs.scale;
    }
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

// head_dim a multiple of 16 (16-byte loads of codes), 16-byte aligned buffers: a thread
// per 16 codes of a K row and the same codes of its V row.  blockIdx.y: (sequence, KV head).
template <typename T, int kFmt>
__global__ void __launch_bounds__(256) kv8_read_vec_kernel(Kv8ReadArgs a, int chunks_per_row) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int bh = blockIdx.y;
    const int b = bh / a.c.n_kv, kvh = bh - b * a.c.n_kv;
    const int it = blockIdx.x * 256 + threadIdx.x;
    const int i = it / chunks_per_row, ch = it - i * chunks_per_row;
    if (i >= a.t) return;
    const int p = a.pos[b] + i;
    size_t row = 0, head_rows = 0;
    bool ok = p >= 0 && p < a.c.max_seq;
    if (!ok && ch == 0) raise_dev_error(kDevErrBadPosition);
    ok = ok && kv8_row(a.c, b, p, row, head_rows, ch == 0);
    row += (size_t)kvh * head_rows;
    uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
    float fk = 0.f, fv = 0.f;
    if (ok) {
        k = ld_stream(a.c.kc + row * a.c.hd + 16 * ch);
        v = ld_stream(a.c.vc + row * a.c.hd + 16 * ch);
        fk = a.c.ks[row];
        fv = a.c.vs[row];
    }
    const size_t o = ((size_t)bh * a.out_rows + i) * a.c.hd + 16 * ch;
    auto expand = [](const uint4& codes, float f, uint16_t* out) {
        const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e += 4) kv8_values4<kFmt>(w[2 * u + e / 4], x + e);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= f;
            *reinterpret_cast<uint4*>(out + 8 * u) = pack8<T>(x);
        }
    };
    expand(k, fk, a.k_out + o);
    expand(v, fv, a.v_out + o);
}

}  // namespace kvb
