// attn_general_src.cuh -- decode attention of any head_dim <= 256 and any group size
// over caches whose rows are found through a source object: the general path behind
// kvb_attention_decode_q8 and kvb_attention_decode_shared.
//
// One warp per (sequence, query head), keys scored 32 at a time (one key per lane),
// the scores folded into an online softmax (running max and sum in f32), each lane
// holding head_dim / 32 output dims.  No key is read twice by a head, but every head
// of a group reads the group's keys: a fallback for shapes and alignments that the
// tensor-core kernels do not take.
#pragma once

#include "kv8.cuh"

namespace kvb {

struct GeneralDecodeArgs {
    const uint16_t* q;
    long long q_row_stride;
    const int32_t* lens;
    int max_len;
    int n_q, n_kv, hd;
    float scale_log2;
    uint16_t* out;
    long long out_row_stride;
};

// 8-bit rows with a scale each.  A row of -1 (a block entry outside the pool) reads as zeros.
template <typename T, int kFmt>
struct Q8Source {
    Kv8Place c;
    __device__ __forceinline__ int keys(int len) const { return len; }
    __device__ __forceinline__ long long row(int b, int kvh, int key) const {
        size_t r, head_rows;
        if (!kv8_row(c, b, key, r, head_rows, true)) return -1;
        return (long long)(r + (size_t)kvh * head_rows);
    }
    __device__ __forceinline__ float dot(long long r, const float* q) const {
        const uint8_t* k = c.kc + (size_t)r * c.hd;
        float s = 0.f;
        for (int d = 0; d < c.hd; ++d) s += q[d] * kv8_value<kFmt>(k[d]);
        return s * c.ks[r];
    }
    __device__ __forceinline__ float v_weight(long long r) const { return c.vs[r]; }
    __device__ __forceinline__ float v(long long r, int d) const {
        return kv8_value<kFmt>(c.vc[(size_t)r * c.hd + d]);
    }
};

// 16-bit rows; keys below `prefix` are the same rows for every sequence.  Contiguous: the
// prefix in pk / pv [n_kv][prefix_rows], own keys in kc / vc.  Paged: everything in the
// pools kc / vc, the prefix through table row 0.
template <typename T>
struct SharedSource {
    const uint16_t* pk;
    const uint16_t* pv;
    int prefix, prefix_rows;
    const uint16_t* kc;
    const uint16_t* vc;
    long long seq_rows;
    int n_kv, hd, max_seq;
    const int32_t* block_table;
    int max_blocks, block_size, n_blocks;
    // paged lengths count the prefix, contiguous ones do not
    __device__ __forceinline__ int keys(int len) const { return block_table ? len : prefix + len; }
    // rows of the prefix buffers are numbered -2 - row
    __device__ __forceinline__ long long row(int b, int kvh, int key) const {
        if (!block_table) {
            if (key < prefix) return -2 - ((long long)kvh * prefix_rows + key);
            return (long long)b * seq_rows + (long long)kvh * max_seq + (key - prefix);
        }
        const int lb = key / block_size;
        const int blk = block_table[(size_t)(key < prefix ? 0 : b) * max_blocks + lb];
        if (blk < 0 || blk >= n_blocks) {
            raise_dev_error(kDevErrBadPosition);
            return -1;
        }
        return ((long long)blk * n_kv + kvh) * block_size + (key - lb * block_size);
    }
    __device__ __forceinline__ float dot(long long r, const float* q) const {
        const T* k = reinterpret_cast<const T*>(r < 0 ? pk : kc) + (size_t)(r < 0 ? -2 - r : r) * hd;
        float s = 0.f;
        for (int d = 0; d < hd; ++d) s += q[d] * Elem<T>::to_f(k[d]);
        return s;
    }
    __device__ __forceinline__ float v_weight(long long) const { return 1.f; }
    __device__ __forceinline__ float v(long long r, int d) const {
        const T* p = reinterpret_cast<const T*>(r < 0 ? pv : vc) + (size_t)(r < 0 ? -2 - r : r) * hd;
        return Elem<T>::to_f(p[d]);
    }
};

template <typename T, class Src>
__global__ void __launch_bounds__(128) attn_general_src_kernel(GeneralDecodeArgs a, Src src) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y * 4 + warp, b = blockIdx.x;
    if (h >= a.n_q) return;
    int len = a.lens[b];
    if (len < 0 || len > a.max_len) {
        if (lane == 0) raise_dev_error(kDevErrBadLength);
        len = len < 0 ? 0 : a.max_len;
    }
    const int n = src.keys(len);
    const int kvh = h / (a.n_q / a.n_kv);
    const T* q = reinterpret_cast<const T*>(a.q) + (size_t)b * a.q_row_stride + (size_t)h * a.hd;
    T* o = reinterpret_cast<T*>(a.out) + (size_t)b * a.out_row_stride + (size_t)h * a.hd;
    __shared__ float qs[4][256];
    for (int d = lane; d < a.hd; d += 32) qs[warp][d] = Elem<T>::to_f(q[d]) * a.scale_log2;
    __syncwarp();
    constexpr int kMaxDims = 8;
    float acc[kMaxDims];
#pragma unroll
    for (int i = 0; i < kMaxDims; ++i) acc[i] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        long long r = -1;
        float s = -INFINITY;
        if (j < n) {
            r = src.row(b, kvh, j);
            s = r == -1 ? 0.f : src.dot(r, qs[warp]);
        }
        const float mn = fmaxf(m, warp_max(s));
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2f(m - ref);
        const float p = j < n ? exp2f(s - ref) : 0.f;
        l = l * alpha + warp_sum(p);
        const float w = r == -1 ? 0.f : p * src.v_weight(r);
#pragma unroll
        for (int i = 0; i < kMaxDims; ++i) acc[i] *= alpha;
        const int nb = min(32, n - j0);
        for (int jj = 0; jj < nb; ++jj) {
            const float pj = __shfl_sync(0xffffffffu, w, jj);
            const long long rj = __shfl_sync(0xffffffffu, r, jj);
            if (rj == -1) continue;
#pragma unroll
            for (int i = 0; i < kMaxDims; ++i) {
                const int d = lane + 32 * i;
                if (d < a.hd) acc[i] += pj * src.v(rj, d);
            }
        }
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < kMaxDims; ++i) {
        const int d = lane + 32 * i;
        if (d < a.hd) o[d] = Elem<T>::from_f(n > 0 ? acc[i] / l : 0.f);
    }
}

}  // namespace kvb
