// attn_decode_q8.cuh -- split-KV GQA decode attention over an 8-bit KV cache, head_dim 64
// or 128, up to 16 query heads per KV head.
//
// Work unit: one CTA per (key chunk, KV head, sequence); its four warps take interleaved
// tiles of 64 keys (head_dim 128: 32), 4 KB of K codes and 4 KB of V codes.  The transposed products put the keys on the MMA's 16-row
// side and the group's heads on its 8-column side, so a group of up to 8 heads wastes no
// rows and takes half the instructions of a 16-row query tile:
//   S^T = K Q^T    A = K codes through ldmatrix (a lane's four bytes are four neighbouring
//                  dims, so that Q's fragments are loaded in that order).  int8: m16n8k32 on the
//                  codes as they are, Q as 16-bit integers in two signed bytes.  e4m3: m16n8k16 on
//                  the codes turned into f16 (exact), Q in f16
//   O^T += V^T P^T m16n8k16, A = V codes as f16 (ldmatrix.trans moves byte pairs: row g of
//                  a tile is dim 2g and row g + 8 is dim 2g + 1), B = P through movmatrix
// int8 codes become f16 through the bytes of 1024 + 128 + code, e4m3 by cvt; both exact.  The
// K scale multiplies the f32 score of its key; the V scale multiplies the key's weight.
// The board's power limit, not HBM, sets the pace of long runs (int8 through f16 for K too:
// 785 us a pass of 256 x 16384 keys at 1470 MHz, 669 us in a burst), so instructions count.
//
// Precision.  Q, int8: round(q * 32639 / max |q|) of the head, in 256 hi + lo, so each element
// is within 1.6e-5 of the head's largest; the products are summed exactly (below 2^31 for
// 128 dims).  Q, e4m3: f16 as it is; bf16 scaled by a power of two to a largest element in
// [2^14, 2^15) and rounded to f16, which is exact for elements down to 2^-31 of the
// largest.  Weights: w = p * v_scale * 2^n, n such that the largest V scale seen makes
// w <= 2^14, rounded once to f16: half a step, 2^-11 of a weight, or 2^-25 where w is below
// 2^-14.  That holds while the V scales, a tile's and those before it, lie in two neighbouring
// magnitudes of 2^8: p = 1 then gives w >= 2^-2, and the second term is at most 2^-23 of such a
// key's weight.  Where they do not (a V row far above the others may have no weight at all), the
// tile's products are f32 multiply-adds on the CUDA cores: 64 x 8 heads x 4096 keys 181 us with
// such a row in every tile, 55 without.
// A remainder as in the 16-bit kernels would double the P V products; the codes
// themselves are within 2^-8 of a row's largest value at best.  Scores, the running
// maximum, the sums and O are f32.
#pragma once

#include "attn_decode.cuh"
#include "kv8.cuh"

namespace kvb {

constexpr int kQ8Warps = 4;
constexpr int kQ8TileBytes = 4096;  // K codes (or V codes) of a tile
constexpr int kQ8Stages = 2;
constexpr int kQ8WarpBytes = kQ8Stages * 2 * kQ8TileBytes;  // a warp's ring: [stage][K | V]
constexpr int kQ8TilesBytes = kQ8Warps * kQ8WarpBytes;
constexpr int kQ8ScaleBytes = kQ8Warps * kQ8Stages * 2 * 64 * 4;
constexpr int kQ8CtasPerSm = 3;
constexpr int kQ8MaxGroup = 16;
constexpr int kQ8SmemBytes = kQ8TilesBytes + kQ8ScaleBytes + 1024;  // with alignment slack

// Floats of one part of the workspace (O, m, l of a group), a multiple of four.
__host__ __device__ constexpr int q8_part_floats(int group, int hd) {
    return (group * (hd + 2) + 3) / 4 * 4;
}
__host__ __device__ constexpr int q8_tile_keys(int hd) { return kQ8TileBytes / hd; }

struct Q8DecodeArgs {
    const uint16_t* q;
    long long q_row_stride;
    const int32_t* lens;
    int max_len, group;
    float scale_log2;
    uint16_t* out;
    long long out_row_stride;
    float* ws;       // split partials: per part O[group][hd], m[group], l[group], padding
    int chunk_keys;  // keys per CTA, a multiple of kQ8Warps tiles
    int max_chunks;
    int piece;       // rows per tensor copy: a whole tile, or gcd(block_size, tile) paged
    int bs_shift;    // paged: log2 of block_size, or -1
    int total_rows;  // rows of the code arrays (a row past the end reads as zeros)
    Kv8Place c;
    // Fused RoPE + append (kRope, kvb_rope_attention_decode_q8): the new token of sequence b is
    // key lens[b] - 1; q points at the qkv rows, unrotated.  Q is rotated in registers, and
    // the CTA of the last chunk quantises the rotated k and the v into that cache row before
    // its tile is requested.
    const float* rope_cos;
    const float* rope_sin;
    int rope_max_pos;
    // kRope: the cache rows before each new key, their scales, the lengths and the block table are
    // final (no kernel that may still be running writes them: the decode-step driver's launches).
    // The first tiles are then requested before griddepcontrol.wait; otherwise nothing is read
    // before it.
    int kv_ready;
};

// One warp's share of the append: a K (rotated) or V row of HD 16-bit elements, quantised to
// codes and scale as kv8_append_vec_kernel does.
template <typename T, int kFmt, int HD>
__device__ __forceinline__ void q8_append_row(const T* in, const float* cos_row, const float* sin_row,
                                              uint8_t* codes, float* scale) {
    constexpr int half = HD / 2;
    const int lane = threadIdx.x & 31;
    float lo[HD / 64], hi[HD / 64];
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
        const int d = lane + 32 * i;
        lo[i] = Elem<T>::to_f(in[d]);
        hi[i] = Elem<T>::to_f(in[d + half]);
        if (cos_row) {
            const float r0 = rot_a(lo[i], hi[i], cos_row[d], sin_row[d]);
            const float r1 = rot_b(lo[i], hi[i], cos_row[d], sin_row[d]);
            lo[i] = Elem<T>::to_f(Elem<T>::from_f(r0));
            hi[i] = Elem<T>::to_f(Elem<T>::from_f(r1));
        }
        mx = max(mx, max(abs_bits(lo[i]), abs_bits(hi[i])));
    }
    const RowScale rs = kv8_row_scale<kFmt>(__reduce_max_sync(0xffffffffu, mx));
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
        const uint32_t c2 = kv8_codes2<kFmt>(lo[i], hi[i], rs.inv);
        codes[lane + 32 * i] = (uint8_t)c2;
        codes[lane + 32 * i + half] = (uint8_t)(c2 >> 8);
    }
    if (lane == 0) *scale = rs.scale;
}

__device__ __forceinline__ int q8_len(const int32_t* lens, int max_len, int b) {
    int len = lens[b];
    if (len < 0 || len > max_len) {
        if (threadIdx.x == 0) raise_dev_error(kDevErrBadLength);
        len = len < 0 ? 0 : max_len;
    }
    return len;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t low16) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}"
        : "=r"(r)
        : "r"(low16));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t v) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
        : "=r"(r)
        : "r"(v));
    return r;
}
// f16 pair of bytes u (codes + 128): 0x64uu is 1024 + u, less 1152 gives the code, exactly.
__device__ __forceinline__ uint32_t biased_to_f16x2(uint32_t u, uint32_t sel) {
    uint32_t r;
    const uint32_t t = prmt(u, 0x64646464u, sel);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(t), "r"(0x64806480u));
    return r;
}
// Four e4m3 codes -> f16 pairs (bytes 0, 1) and (2, 3).
__device__ __forceinline__ void codes_pairs(uint32_t v, uint32_t& p01, uint32_t& p23) {
    p01 = e4m3x2_to_f16x2(v);
    p23 = e4m3x2_hi_to_f16x2(v);
}
// Four codes -> f16 pairs (bytes 0, 2) and (1, 3).
template <int kFmt>
__device__ __forceinline__ void codes_evens_odds(uint32_t v, uint32_t& p02, uint32_t& p13) {
    if (kFmt == KVB_KV_INT8) {
        const uint32_t u = v ^ 0x80808080u;
        p02 = biased_to_f16x2(u, 0x4240u);
        p13 = biased_to_f16x2(u, 0x4341u);
    } else {
        const uint32_t u = prmt(v, 0u, 0x3120u);
        p02 = e4m3x2_to_f16x2(u);
        p13 = e4m3x2_hi_to_f16x2(u);
    }
}
// D (s32) += A (16 x 32, s8) B (32 x 8, s8)
__device__ __forceinline__ void mma_s8(int* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                       uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9},"
        " {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Low bytes of four integers, in order.
__device__ __forceinline__ uint32_t bytes4(int a, int b, int c, int d) {
    return prmt(prmt((uint32_t)a, (uint32_t)b, 0x0040u), prmt((uint32_t)c, (uint32_t)d, 0x0040u),
                0x5410u);
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 4-byte asynchronous copy to shared memory; bytes == 0 writes zero and reads nothing.
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
}
// Arrives on the barrier once this thread's earlier cp.async copies have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// Magnitude of a V scale: bit i for exponents 8 i .. 8 i + 7 (2^(8 i + 8 - 127) itself included,
// 2^(8 i - 127) not); no bit for 0, whose shift is beyond 31.
__device__ __forceinline__ uint32_t mag_bit(float scale) {
    uint32_t r;
    asm("shl.b32 %0, %1, %2;" : "=r"(r) : "r"(1u), "r"((abs_bits(scale) - 1u) >> 26));
    return r;
}
// 2^(133 - 8 i): takes magnitude i (1 .. 31) to 2^14 at most.
__device__ __forceinline__ float q8_v_factor(int i) {
    return __uint_as_float((uint32_t)(260 - 8 * i) << 23);
}
// to / from, powers of two, or 0 where that is below f32's normal numbers.
__device__ __forceinline__ float q8_v_rescale(float from, float to) {
    const int e = 127 + (int)(__float_as_uint(to) >> 23) - (int)(__float_as_uint(from) >> 23);
    return e > 0 ? __uint_as_float((uint32_t)e << 23) : 0.f;
}

// Byte offset of 16-byte chunk `ch` of row r in a tile that the tensor copy wrote with a
// 64-byte (head_dim 64) or 128-byte swizzle.
template <int HD>
__device__ __forceinline__ uint32_t q8_smem_off(int r, int ch) {
    return HD == 64 ? (uint32_t)(r * 64 + ((ch ^ ((r >> 1) & 3)) << 4))
                    : (uint32_t)(r * 128 + ((ch ^ (r & 7)) << 4));
}

// Grid (KV head, sequence, chunk slot); slots count chunks from the end of the sequence, so full
// chunks are dispatched first (as attn_decode.cuh).
template <typename T, int kFmt, int HD, int NT, bool kRope>
__global__ void __launch_bounds__(128, kQ8CtasPerSm)
    attn_decode_q8_kernel(const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap, Q8DecodeArgs a) {
    constexpr int KT = q8_tile_keys(HD);  // keys per tile
    constexpr int MT = KT / 16;           // 16-key MMA rows of S^T, k-steps of P V
    constexpr int DT = HD / 16;           // 16-dim chunks: k-steps of K Q, MMA rows of O^T
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[kQ8Warps][kQ8Stages][2];  // K tile and scales; V tile and scales
    __shared__ float w_ml[kQ8Warps][2][kQ8MaxGroup];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    const int kvh = blockIdx.x, b = blockIdx.y;
    const int G = a.group;
    if (threadIdx.x < kQ8Warps * kQ8Stages * 2)
        mbar_init(&bars[0][0][0] + threadIdx.x, 1 + 32);  // one expect_tx, 32 scale arrivals
    fence_mbar_init();
    __syncthreads();
    const bool early = kRope && a.kv_ready;
    // The join may start once every CTA has waited: the lengths, which an earlier kernel may have
    // written, are then final for it.
    auto wait = [] {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;");
    };
    if (!early) wait();

    const int len = q8_len(a.lens, a.max_len, b);
    const int n_chunks = (len + a.chunk_keys - 1) / a.chunk_keys;
    const int from_end = a.max_chunks - 1 - (int)blockIdx.z;
    T* outb = reinterpret_cast<T*>(a.out) + (size_t)b * a.out_row_stride + (size_t)kvh * G * HD;
    if (len == 0) {  // no keys: a zero row
        if (early) wait();
        if (from_end == 0)
            for (int i = threadIdx.x; i < G * HD; i += blockDim.x) outb[i] = Elem<T>::from_f(0.f);
        return;
    }
    if (from_end >= n_chunks) return;
    uint8_t* ring = smem + warp * kQ8WarpBytes;
    float* ring_scales = reinterpret_cast<float*>(smem + kQ8TilesBytes) + warp * kQ8Stages * 128;
    // this warp's O for the merge, [8 NT][HD] over its own tiles
    float* wo = reinterpret_cast<float*>(ring);
    const int chunk = n_chunks - 1 - from_end;
    const int key_begin = chunk * a.chunk_keys;
    const int key_end = min(len, key_begin + a.chunk_keys);
    const int row_base = (int)(b * a.c.seq_rows + (long long)kvh * a.c.max_seq);
    const int pshift = __ffs(a.piece) - 1;
    // The new token's position (-1: none, or outside the tables or the cache).  A length past
    // max_len is clamped for the attention alone: row max_len - 1 holds another token.
    int rope_p = -1;
    if (kRope) {
        rope_p = a.lens[b] - 1;
        if (rope_p >= a.rope_max_pos || rope_p >= a.c.max_seq) {
            if (threadIdx.x == 0) raise_dev_error(kDevErrBadPosition);
            rope_p = -1;
        }
    }
    const bool appends = kRope && rope_p >= 0 && chunk == n_chunks - 1;  // CTA-uniform

    // Paged: this lane's piece of the next tile to be requested, read a tile ahead.
    auto block_of = [&](int kt0) -> int {
        const int k = kt0 + (lane << pshift);
        if (!a.c.block_table || lane >= (KT >> pshift) || k >= key_end) return 0;
        const int lb = a.bs_shift >= 0 ? k >> a.bs_shift : k / a.c.block_size;
        return a.c.block_table[(size_t)b * a.c.max_blocks + lb];
    };
    int blk = block_of(key_begin + warp * KT);
    // The tile that is requested next: its pieces, this lane's piece's row, and the rows of
    // this lane's two keys (-1: none, their scales are zero).
    int n_pieces = 0, row = 0, key_row[KT / 32];
    auto place = [&](int kt0) {
        const int nk = min(KT, key_end - kt0);
        if (!a.c.block_table) {
            n_pieces = 1;
            row = row_base + kt0;
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
                key_row[u] = lane + 32 * u < nk ? row + lane + 32 * u : -1;
            return;
        }
        n_pieces = (nk + a.piece - 1) >> pshift;
        row = a.total_rows;  // past the end: zeros
        if (lane < n_pieces) {
            if (blk < 0 || blk >= a.c.n_blocks)
                raise_dev_error(kDevErrBadPosition);
            else {
                const int k = kt0 + (lane << pshift);
                row = (blk * a.c.n_kv + kvh) * a.c.block_size +
                      (a.bs_shift >= 0 ? k & (a.c.block_size - 1) : k % a.c.block_size);
            }
        }
        blk = block_of(kt0 + kQ8Warps * KT);  // of the tile that is placed next
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) {
            const int k = lane + 32 * u;
            const int r0 = __shfl_sync(0xffffffffu, row, k >> pshift);
            key_row[u] = k < nk && r0 < a.total_rows ? r0 + (k & (a.piece - 1)) : -1;
        }
    };
    // Requests the placed tile's K (or V) codes by tensor copies and scales by 4-byte
    // copies, all counted on the tile's barrier.
    auto request = [&](const CUtensorMap& map, uint8_t* tile, const float* scales, float* dst,
                       uint64_t* bar) {
        if (lane == 0) mbar_expect_tx(bar, (uint32_t)(n_pieces * a.piece * HD));
        __syncwarp();
        if (lane < n_pieces) tma_load_2d(tile + (lane << pshift) * HD, &map, bar, 0, row);
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
            cp_async4(smem_u32(dst + lane + 32 * u), scales + max(key_row[u], 0),
                      key_row[u] >= 0 ? 4 : 0);
        cp_async_arrive(bar);
    };
    auto request_k = [&](int st) {
        request(kmap, ring + st * 2 * kQ8TileBytes, a.c.ks, ring_scales + st * 128,
                &bars[warp][st][0]);
    };
    auto request_v = [&](int st) {
        request(vmap, ring + (st * 2 + 1) * kQ8TileBytes, a.c.vs, ring_scales + st * 128 + 64,
                &bars[warp][st][1]);
    };
    // The first tiles; the one that holds the new key waits until that row is written (it is
    // its warp's last).
    auto first_tiles = [&](bool holding) {
#pragma unroll
        for (int i = 0; i < kQ8Stages; ++i) {
            const int kt0 = key_begin + (warp + i * kQ8Warps) * KT;
            if (kt0 < key_end && (appends && rope_p < kt0 + KT) == holding) {
                place(kt0);
                request_k(i);
                request_v(i);
            }
        }
    };
    first_tiles(false);
    if (early) wait();  // q, the new row
    if (appends) {
        size_t crow = 0, head_rows = 0;
        if (warp < 2 && kv8_row(a.c, b, rope_p, crow, head_rows, threadIdx.x == 0)) {
            crow += (size_t)kvh * head_rows;
            const T* in = reinterpret_cast<const T*>(a.q) + (size_t)b * a.q_row_stride +
                          (size_t)(a.c.n_kv * (G + warp) + kvh) * HD;
            if (warp == 0)
                q8_append_row<T, kFmt, HD>(in, a.rope_cos + (size_t)rope_p * (HD / 2),
                                           a.rope_sin + (size_t)rope_p * (HD / 2),
                                           a.c.kc + crow * HD, a.c.ks + crow);
            else
                q8_append_row<T, kFmt, HD>(in, nullptr, nullptr, a.c.vc + crow * HD, a.c.vs + crow);
        }
        // the tensor copies read these rows through the async proxy
        asm volatile("fence.proxy.async.global;" ::: "memory");
        __syncthreads();
        first_tiles(true);
    }

    // Q fragments (B operand): column g = head 8 nt + g, dims 16 j + 4c .. + 3.  int8: the
    // high bytes, then the low ones; e4m3: two f16 pairs.
    uint32_t qf[DT][NT][2];
    float qs[NT][2];  // score factor of heads 8 nt + 2c, + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int h = 8 * nt + g;
        const T* qr = reinterpret_cast<const T*>(a.q) + (size_t)b * a.q_row_stride +
                      (size_t)(kvh * G + min(h, G - 1)) * HD;
        uint2 v[DT];
#pragma unroll
        for (int j = 0; j < DT; ++j)
            v[j] = h < G ? *reinterpret_cast<const uint2*>(qr + 16 * j + 4 * c) : make_uint2(0u, 0u);
        if (kRope && rope_p >= 0) {
            // rotate_half in registers: chunk j pairs with chunk j + DT / 2, the same lane
#pragma unroll
            for (int j = 0; j < DT / 2; ++j) {
                const size_t at = (size_t)rope_p * (HD / 2) + 16 * j + 4 * c;
                const float4 cs = *reinterpret_cast<const float4*>(a.rope_cos + at);
                const float4 sn = *reinterpret_cast<const float4*>(a.rope_sin + at);
                auto rotate2 = [](uint32_t& lo, uint32_t& hi, float c0, float c1, float s0, float s1) {
                    const float2 x = Elem<T>::unpack(lo), y = Elem<T>::unpack(hi);
                    lo = Elem<T>::pack(rot_a(x.x, y.x, c0, s0), rot_a(x.y, y.y, c1, s1));
                    hi = Elem<T>::pack(rot_b(x.x, y.x, c0, s0), rot_b(x.y, y.y, c1, s1));
                };
                rotate2(v[j].x, v[j + DT / 2].x, cs.x, cs.y, sn.x, sn.y);
                rotate2(v[j].y, v[j + DT / 2].y, cs.z, cs.w, sn.z, sn.w);
            }
        }
        float f = a.scale_log2;
        if (kFmt == KVB_KV_INT8) {
            uint32_t mx = 0;  // the head's largest magnitude, as a bit pattern
#pragma unroll
            for (int j = 0; j < DT; ++j) {
                const float2 x = Elem<T>::unpack(v[j].x), y = Elem<T>::unpack(v[j].y);
                mx = max(max(mx, max(abs_bits(x.x), abs_bits(x.y))),
                         max(abs_bits(y.x), abs_bits(y.y)));
            }
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float big = fmaxf(__uint_as_float(mx), 0x1p-100f);
            const float up = __fdiv_rn(32639.f, big);
            // a NaN or an infinity among the elements: every score of the head is NaN
            f = mx < 0x7f800000u ? f * __fdiv_rn(big, 32639.f) : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int j = 0; j < DT; ++j) {
                const float2 x = Elem<T>::unpack(v[j].x), y = Elem<T>::unpack(v[j].y);
                const int i0 = __float2int_rn(x.x * up), i1 = __float2int_rn(x.y * up);
                const int i2 = __float2int_rn(y.x * up), i3 = __float2int_rn(y.y * up);
                v[j].x = bytes4((i0 + 128) >> 8, (i1 + 128) >> 8, (i2 + 128) >> 8, (i3 + 128) >> 8);
                v[j].y = bytes4(i0, i1, i2, i3);  // i - 256 hi, in -128 .. 127
            }
        } else if (Elem<T>::kDtype == KVB_BF16) {
            uint32_t mx = 0;  // largest exponent of the head's elements
#pragma unroll
            for (int j = 0; j < DT; ++j)
                mx = max(max(mx, max(v[j].x & 0x7fffu, (v[j].x >> 16) & 0x7fffu)),
                         max(v[j].y & 0x7fffu, (v[j].y >> 16) & 0x7fffu));
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // biased exponent, kept where 2^(14 - e) and its inverse are normal numbers
            const int e = min(max((int)(mx >> 7), 16), 254);
            const float up = __uint_as_float((uint32_t)(268 - e) << 23);  // 2^(141 - e)
            f *= __uint_as_float((uint32_t)(e - 14) << 23);               // 2^(e - 141)
#pragma unroll
            for (int j = 0; j < DT; ++j) {
                const float2 x = Elem<T>::unpack(v[j].x), y = Elem<T>::unpack(v[j].y);
                v[j].x = f16x2(x.x * up, x.y * up);
                v[j].y = f16x2(y.x * up, y.y * up);
            }
        }
#pragma unroll
        for (int j = 0; j < DT; ++j) {
            qf[j][nt][0] = v[j].x;
            qf[j][nt][1] = v[j].y;
        }
        qs[nt][0] = __shfl_sync(0xffffffffu, f, 8 * c);
        qs[nt][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
    }

    float o[DT][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < DT; ++j) o[j][nt][0] = o[j][nt][1] = o[j][nt][2] = o[j][nt][3] = 0.f;
    }
    // Magnitudes (eighths of the exponent range, a bit each) of the V scales so far, two
    // neighbours at most; O is in units of 1 / vf, the factor that takes the upper one below 2^14.
    uint32_t seen = 0;
    float vf = q8_v_factor(1);
    // Two tiles per warp in flight, K and V on barriers of their own: the K of the tile
    // after next is requested once the scores are out of this one, its V once P V has read
    // this V.
    bool ok = true;
    int it = 0;
    bool k_failed = false;
    for (int kt0 = key_begin + warp * KT; kt0 < key_end; kt0 += kQ8Warps * KT, ++it) {
        const int st = it % kQ8Stages;
        const uint32_t phase = (it / kQ8Stages) & 1;
        const int nk = min(KT, key_end - kt0);
        const int kt_next = kt0 + kQ8Stages * kQ8Warps * KT;
        const bool more = kt_next < key_end;
        const uint32_t kb = smem_u32(ring + st * 2 * kQ8TileBytes), vb = kb + kQ8TileBytes;
        const float* ks = ring_scales + st * 128;
        const float* vs = ks + 64;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars[warp][st][0], phase));
        if (!ok) {
            k_failed = true;
            break;
        }

        // ---- S^T = K Q^T
        float s[MT][NT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = 16 * t + (lane & 15);
            if constexpr (kFmt == KVB_KV_INT8) {
                int hi[NT][4], lo[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) hi[nt][e] = lo[nt][e] = 0;
#pragma unroll
                for (int j = 0; j < DT; j += 2) {
                    uint32_t w0, w1, w2, w3;
                    ldsm_x4(kb + q8_smem_off<HD>(r, j + (lane >> 4)), w0, w1, w2, w3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_s8(hi[nt], w0, w1, w2, w3, qf[j][nt][0], qf[j + 1][nt][0]);
                        mma_s8(lo[nt], w0, w1, w2, w3, qf[j][nt][1], qf[j + 1][nt][1]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][nt][e] = (float)(hi[nt][e] * 256 + lo[nt][e]);
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    s[t][nt][0] = s[t][nt][1] = s[t][nt][2] = s[t][nt][3] = 0.f;
#pragma unroll
                for (int j = 0; j < DT; j += 2) {
                    uint32_t w0, w1, w2, w3, af[4];
                    ldsm_x4(kb + q8_smem_off<HD>(r, j + (lane >> 4)), w0, w1, w2, w3);
                    codes_pairs(w0, af[0], af[2]);
                    codes_pairs(w1, af[1], af[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_16816<__half>(s[t][nt], af, qf[j][nt][0], qf[j][nt][1]);
                    codes_pairs(w2, af[0], af[2]);
                    codes_pairs(w3, af[1], af[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_16816<__half>(s[t][nt], af, qf[j + 1][nt][0], qf[j + 1][nt][1]);
                }
            }
        }
        // ---- scale and mask; element e: key 16 t + g + 8 (e >> 1), head 8 nt + 2c + (e & 1)
        float mx[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float k0 = ks[16 * t + g], k1 = ks[16 * t + g + 8];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][nt][e] *= (e < 2 ? k0 : k1) * qs[nt][e & 1];
        }
        __syncwarp();
        fence_async_smem();  // these reads precede the next copies into the K tile
        if (more) {
            place(kt_next);
            request_k(st);
        }
        if (nk < KT) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (16 * t + g + 8 * (e >> 1) >= nk) s[t][nt][e] = -INFINITY;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                mx[nt][0] = fmaxf(mx[nt][0], fmaxf(s[t][nt][0], s[t][nt][2]));
                mx[nt][1] = fmaxf(mx[nt][1], fmaxf(s[t][nt][1], s[t][nt][3]));
            }
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                mx[nt][0] = fmaxf(mx[nt][0], __shfl_xor_sync(0xffffffffu, mx[nt][0], x));
                mx[nt][1] = fmaxf(mx[nt][1], __shfl_xor_sync(0xffffffffu, mx[nt][1], x));
            }
        }
        float al[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float mn = fmaxf(m[nt][e], mx[nt][e]);
                const float ref = mn == -INFINITY ? 0.f : mn;
                al[nt][e] = ex2_approx(m[nt][e] - ref);
                m[nt][e] = mn;
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    s[t][nt][e] = ex2_approx(s[t][nt][e] - ref);
                    s[t][nt][e + 2] = ex2_approx(s[t][nt][e + 2] - ref);
                    sum += s[t][nt][e] + s[t][nt][e + 2];
                }
                // this lane's keys; summed over lanes at the end
                l[nt][e] = l[nt][e] * al[nt][e] + sum;
            }
        ok = __all_sync(0xffffffffu, mbar_wait(&bars[warp][st][1], phase));
        if (!ok) break;
        if (kFmt == KVB_KV_E4M3 && nk < KT) {  // codes past the last key may be NaN: 0 * NaN
            for (int i = nk * HD / 16 + lane; i < KT * HD / 16; i += 32)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vb + 16 * i), "r"(0)
                             : "memory");
            __syncwarp();
        }
        // ---- V scale magnitudes: O is rescaled where larger ones appear.  (The first V fragment
        // is read beside them: the check costs 0.8 % of a long pass, 2.3 % with its latency bare.)
        uint32_t first[4];
        ldsm_x4_t(vb + q8_smem_off<HD>(lane & 15, lane >> 4), first[0], first[1], first[2], first[3]);
        uint32_t mags = mag_bit(vs[lane]);
        if (KT == 64) mags |= mag_bit(vs[lane + 32]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < DT; ++j) {
                    o[j][nt][e] *= al[nt][e];
                    o[j][nt][e + 2] *= al[nt][e];
                }
        float vt = vf;  // the MMA's factor: 0 where the tile is done without it
        if (__any_sync(0xffffffffu, mags & ~seen)) {
            // (A row with a NaN makes every head NaN as it is, and has no magnitude.)
            mags = abs_bits(vs[lane]) < 0x7f800000u ? mag_bit(vs[lane]) : 0u;
            if (KT == 64 && abs_bits(vs[lane + 32]) < 0x7f800000u) mags |= mag_bit(vs[lane + 32]);
            mags = __reduce_or_sync(0xffffffffu, mags) | seen;
            auto rescale = [&](float r) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < DT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[j][nt][e] *= r;
            };
            const int top = max(31 - __clz(mags), 1);
            float r = 1.f;  // 2^ of the change of O's unit
            if (mags & ~(3u << (top - 1))) {
                // Far apart: w = p * scale in f32, its largest sets the unit, and the products
                // are multiply-adds.
                uint32_t wmax = 0;
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[t][nt][e] *= vs[16 * t + g + 8 * (e >> 1)];
                            const uint32_t w = abs_bits(s[t][nt][e]);
                            if (w < 0x7f800000u) wmax = max(wmax, w);
                        }
                const int wtop = max((int)(__reduce_max_sync(0xffffffffu, wmax) >> 26), 1);
                if (q8_v_factor(wtop) < vf) {
                    r = q8_v_rescale(vf, q8_v_factor(wtop));
                    vf = q8_v_factor(wtop);
                    seen = 1u << wtop;
                }
                rescale(r);
#pragma unroll 1
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int t = 0; t < 2 * MT; ++t) {  // key 8 t + i: its weights are in row i's lanes
                        float w[NT][2];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                w[nt][e] = vf * __shfl_sync(0xffffffffu, s[t / 2][nt][2 * (t % 2) + e],
                                                            4 * i + c);
#pragma unroll
                        for (int j = 0; j < DT; ++j) {
                            uint16_t v;
                            asm volatile("ld.shared.u16 %0, [%1];"
                                         : "=h"(v)
                                         : "r"(vb + q8_smem_off<HD>(8 * t + i, j) + 2 * g));
                            const float x0 = kv8_value<kFmt>((uint8_t)v);
                            const float x1 = kv8_value<kFmt>((uint8_t)(v >> 8));
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    o[j][nt][e] += w[nt][e] * x0;
                                    o[j][nt][e + 2] += w[nt][e] * x1;
                                }
                        }
                    }
                vt = 0.f;
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        s[t][nt][0] = s[t][nt][1] = s[t][nt][2] = s[t][nt][3] = 0.f;
            } else {
                if (q8_v_factor(top) < vf) {
                    r = q8_v_rescale(vf, q8_v_factor(top));
                    vf = q8_v_factor(top);
                }
                seen = mags;
                vt = vf;
                rescale(r);
            }
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float v0 = vs[16 * t + g] * vt, v1 = vs[16 * t + g + 8] * vt;
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                pf[nt][0] = movmatrix_t(f16x2(s[t][nt][0] * v0, s[t][nt][1] * v0));
                pf[nt][1] = movmatrix_t(f16x2(s[t][nt][2] * v1, s[t][nt][3] * v1));
            }
            const int r = 16 * t + (lane & 15);
#pragma unroll
            for (int j = 0; j < DT; j += 2) {
                uint32_t w0, w1, w2, w3, af[4];
                if (t == 0 && j == 0) {
                    w0 = first[0];
                    w1 = first[1];
                    w2 = first[2];
                    w3 = first[3];
                } else {
                    ldsm_x4_t(vb + q8_smem_off<HD>(r, j + (lane >> 4)), w0, w1, w2, w3);
                }
                codes_evens_odds<kFmt>(w0, af[0], af[1]);
                codes_evens_odds<kFmt>(w1, af[2], af[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816<__half>(o[j][nt], af, pf[nt][0], pf[nt][1]);
                codes_evens_odds<kFmt>(w2, af[0], af[1]);
                codes_evens_odds<kFmt>(w3, af[2], af[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_16816<__half>(o[j + 1][nt], af, pf[nt][0], pf[nt][1]);
            }
        }
        __syncwarp();
        fence_async_smem();  // these reads precede the next copies into the V tile
        if (more) request_v(st);
    }
    if (!ok) {
        // A copy did not complete in time (the error word is set): wait once more, bounded,
        // for each copy still outstanding, and contribute an empty state.
        for (int i = it; i <= it + kQ8Stages; ++i) {
            if (key_begin + (warp + i * kQ8Warps) * KT >= key_end) break;
            const uint32_t ph = (i / kQ8Stages) & 1;
            const bool k_asked = i < it + kQ8Stages || !k_failed;
            if (k_asked && (i > it || k_failed)) mbar_wait(&bars[warp][i % kQ8Stages][0], ph);
            if (i < it + kQ8Stages) mbar_wait(&bars[warp][i % kQ8Stages][1], ph);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int j = 0; j < DT; ++j) o[j][nt][0] = o[j][nt][1] = o[j][nt][2] = o[j][nt][3] = 0.f;
        }
        __syncwarp();
    }
    // ---- merge the four warps' states through shared memory
    const float unit = __uint_as_float((254u << 23) - __float_as_uint(vf));  // 1 / vf, a power of two
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
            const int h = 8 * nt + 2 * c + e;
            if (g == 0) {
                w_ml[warp][0][h] = m[nt][e];
                w_ml[warp][1][h] = l[nt][e];
            }
#pragma unroll
            for (int j = 0; j < DT; ++j)
                *reinterpret_cast<float2*>(wo + h * HD + 16 * j + 2 * g) =
                    make_float2(o[j][nt][e] * unit, o[j][nt][e + 2] * unit);
        }
    }
    __syncthreads();
    float* wsb = nullptr;
    if (n_chunks > 1)
        wsb = a.ws + (((size_t)b * a.c.n_kv + kvh) * a.max_chunks + chunk) *
                         (size_t)q8_part_floats(G, HD);
    // Four neighbouring dims of one head per thread and turn; 128 threads span 512 / HD
    // heads a turn.
    for (int i = 4 * threadIdx.x; i < G * HD; i += 4 * kQ8Warps * 32) {
        const int r = i / HD;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kQ8Warps; ++w) M = fmaxf(M, w_ml[w][0][r]);
        float L = 0.f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kQ8Warps; ++w) {
            const float mw = w_ml[w][0][r];
            const float f = mw == -INFINITY ? 0.f : ex2_approx(mw - M);
            // a warp whose scores were all NaN keeps -inf as its maximum and a NaN sum
            const float lw = w_ml[w][1][r];
            L += lw != lw ? lw : lw * f;
            const float4 ow = *reinterpret_cast<const float4*>(smem + w * kQ8WarpBytes + 4 * i);
            O.x += ow.x * f;
            O.y += ow.y * f;
            O.z += ow.z * f;
            O.w += ow.w * f;
        }
        if (n_chunks == 1) {
            const float inv = 1.f / L;
            outb[i] = Elem<T>::from_f(O.x * inv);
            outb[i + 1] = Elem<T>::from_f(O.y * inv);
            outb[i + 2] = Elem<T>::from_f(O.z * inv);
            outb[i + 3] = Elem<T>::from_f(O.w * inv);
        } else {
            *reinterpret_cast<float4*>(wsb + i) = O;
            if (i % HD == 0) {
                wsb[G * HD + r] = M;
                wsb[G * HD + G + r] = L;
            }
        }
    }
}

// Joins the partial states of every (sequence, head): parts 0 .. fixed - 1, which every
// sequence has, then one for each chunk of its keys past own_key0.  Written rows: those with more
// than one part (write_all: every row, zeros where a sequence has no keys).  A row that has keys
// but no score above -infinity is 0 / 0, as it is in one chunk.  A programmatic
// dependent of the kernel that writes the partials.  Latency bounds it, so a row is one warp's (or
// W of its CTA's eight, parts w, w + W, ..., where there are more than 32): the lanes are laid
// out as (part, four neighbouring outputs), each requests its first kAhead parts' O, 16 bytes
// a load, beside the parts' (m, l), a part a lane, so that all reads share one latency and
// nothing goes through shared memory.  Parts start on 16 bytes.  Measured in the calls that end
// with it: 256 sequences x 32 heads of 9 parts 59.6 us, where a CTA per (sequence, KV head) with
// the weights in shared memory took 64.5; 37 x 16 heads of 128 dims, 18.0 against 19.7.  16 loads
// ahead instead of 8 where 8 reach all parts cost the many rows residency (62.1 us); where they
// do not, 2048 rows of 18 parts: 22.0 us, two warps of 8 ahead 23.8, one of 8 ahead 23.7.
struct JoinArgs {
    const float* ws;
    const int32_t* lens;
    int max_len, key0, chunk_keys;
    int fixed, max_parts, part_floats;
    int n_kv, group;
    int write_all;
    int prefix;  // keys of every sequence that its length does not count
    uint16_t* out;
    long long out_row_stride;
};
constexpr int kJoinWarps = 8;
constexpr int kJoinMaxParts = 512;
// Grid (groups of kJoinWarps / W heads, sequence).
template <typename T, int HD, int W, int kAhead>
__global__ void __launch_bounds__(32 * kJoinWarps) attn_join_kernel(JoinArgs a) {
    constexpr int kCols = HD / 4, kLanes = 32 / kCols;  // lanes of a row, parts side by side
    __shared__ float ml[kJoinWarps][2];
    __shared__ float4 sums[W > 1 ? kJoinWarps : 1][kCols];
    asm volatile("griddepcontrol.launch_dependents;");
    // What the lengths come from has completed when this grid starts; the partials have not.
    int len = ld_from<true>(a.lens + blockIdx.y);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.group, b = blockIdx.y, n_q = a.n_kv * G;
    const int w = warp % W;
    const int head = blockIdx.x * (kJoinWarps / W) + warp / W;
    const bool have = head < n_q;
    const int kvh = min(head, n_q - 1) / G, r = min(head, n_q - 1) - kvh * G;
    const int per4 = a.part_floats / 4;
    const float* base = a.ws + ((size_t)b * a.n_kv + kvh) * a.max_parts * (size_t)a.part_floats;
    const float4* o4 = reinterpret_cast<const float4*>(base + r * HD) + lane % kCols;
    const int side = lane / kCols;
    // this warp's parts: w + W q
    auto part = [&](int q) { return w + W * q; };
    if (len < 0 || len > a.max_len) {
        if (threadIdx.x == 0) raise_dev_error(kDevErrBadLength);
        len = len < 0 ? 0 : a.max_len;
    }
    const int own = (len - own_key0(len, a.key0) + a.chunk_keys - 1) / a.chunk_keys;
    const int parts = a.fixed + own;
    if (!a.write_all && parts <= 1) return;  // the same for the whole CTA
    float4 ahead[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        const int p = part(kLanes * k + side);
        ahead[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p < parts) ahead[k] = o4[(size_t)p * per4];
    }
    float M = -INFINITY, L = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    // a part without weight may hold anything (0 * NaN where every key was masked)
    auto add = [&](const float4& o, float f) {
        if (f == 0.f) return;
        x.x += o.x * f;
        x.y += o.y * f;
        x.z += o.z * f;
        x.w += o.w * f;
    };
    auto rescale = [&](float f) {
        x.x *= f;
        x.y *= f;
        x.z *= f;
        x.w *= f;
    };
    for (int q0 = 0; part(q0) < parts; q0 += 32) {  // 32 parts at a time, one per lane
        const int p = part(q0 + lane);
        float mp = -INFINITY, lp = 0.f;
        if (p < parts) {
            mp = base[(size_t)p * a.part_floats + G * HD + r];
            lp = base[(size_t)p * a.part_floats + G * HD + G + r];
        }
        const float Mn = fmaxf(M, warp_max(mp));
        const float f = mp == -INFINITY ? 0.f : exp2f(mp - Mn);
        const float down = M == -INFINITY ? 0.f : exp2f(M - Mn);
        if (q0 > 0) {
            L *= down;
            if (M != Mn) rescale(down);
        }
        M = Mn;
        L += warp_sum(lp != lp ? lp : lp * f);
#pragma unroll
        for (int k = 0; k < 32 / kLanes; ++k) {
            const int q = kLanes * k + side;
            const float fq = __shfl_sync(0xffffffffu, f, q);
            if (part(q0 + kLanes * k) >= parts) break;
            if (k < kAhead && q0 == 0) add(ahead[k < kAhead ? k : 0], fq);
            else if (part(q0 + q) < parts) add(o4[(size_t)part(q0 + q) * per4], fq);
        }
    }
    if (kLanes == 2) {  // the two sides' parts
        x.x += __shfl_xor_sync(0xffffffffu, x.x, 16);
        x.y += __shfl_xor_sync(0xffffffffu, x.y, 16);
        x.z += __shfl_xor_sync(0xffffffffu, x.z, 16);
        x.w += __shfl_xor_sync(0xffffffffu, x.w, 16);
    }
    if constexpr (W > 1) {
        if (lane == 0) {
            ml[warp][0] = M;
            ml[warp][1] = L;
        }
        if (lane < kCols) sums[warp][lane] = x;
        __syncthreads();
        if (w != 0) return;
        float Mr = -INFINITY;
#pragma unroll
        for (int i = 0; i < W; ++i) Mr = fmaxf(Mr, ml[warp + i][0]);
        L = 0.f;
        x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float f = ml[warp + i][0] == -INFINITY ? 0.f : exp2f(ml[warp + i][0] - Mr);
            const float li = ml[warp + i][1];
            L += li != li ? li : li * f;
            add(sums[warp + i][lane % kCols], f);
        }
    }
    if (!have || lane >= kCols) return;
    const float inv = len + a.prefix > 0 ? 1.f / L : 0.f;
    T* out = reinterpret_cast<T*>(a.out) + (size_t)b * a.out_row_stride + (size_t)head * HD + 4 * lane;
    if ((reinterpret_cast<uintptr_t>(out) & 7) == 0) {
        *reinterpret_cast<uint2*>(out) = make_uint2(Elem<T>::pack(x.x * inv, x.y * inv),
                                                    Elem<T>::pack(x.z * inv, x.w * inv));
    } else {
        out[0] = Elem<T>::from_f(x.x * inv);
        out[1] = Elem<T>::from_f(x.y * inv);
        out[2] = Elem<T>::from_f(x.z * inv);
        out[3] = Elem<T>::from_f(x.w * inv);
    }
}

}  // namespace kvb
