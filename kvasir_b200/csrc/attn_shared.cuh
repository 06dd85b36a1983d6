// attn_shared.cuh -- decode attention of many sequences over one shared prefix, on the
// 5th-generation tensor cores (tcgen05 / TMEM), head_dim 64.
//
// A decode step reads every key once per sequence.  Where sequences share their first
// keys, those are read once for all of them: the query rows of the sequences that share
// a KV head (n_seq x n_q / n_kv rows) become the 128 rows of an MMA tile, which turns the
// prefix's part of the step from a stream of K and V per sequence into a matrix product.
// One CTA computes one tile of 128 / group sequences x group heads against one slice of
// the prefix and writes an unnormalised partial (O, running max, sum) per row; the own
// keys of each sequence go through the split-KV decode kernel, which writes partials of
// the same form, and attn_join_kernel joins them.
//
// The pipeline is attn_prefill.cuh's (its comments give the reasons): warp 4 brings Q once
// and 96-key K/V tiles through a 3-stage ring, warp 5 issues S = Q K^T and O += P V with P
// in TMEM, warps 0-3 hold one row per thread; two CTAs share an SM.  There is no causal
// mask; a row's keys end at the prefix's end, or earlier for a paged sequence shorter
// than the prefix.
#pragma once

#include "attn_decode_q8.cuh"
#include "attn_prefill.cuh"

namespace kvb {

struct SharedPrefixArgs {
    int n_seq, n_kv, group, seqs_per_tile;
    int prefix;           // keys of the prefix
    int n_tiles, splits;  // 96-key tiles of the prefix, slices they are dealt to
    float scale_log2;
    const int32_t* lens;  // paged: lengths that may end inside the prefix; else nullptr
    int max_len;
    float* ws;  // partials [n_seq][n_kv][max_parts][group * 66]; slice i is part i
    int max_parts;
    const int32_t* block_table;  // row 0 holds the prefix's blocks; nullptr = contiguous
    int block_size, n_blocks;
};

template <typename T>
__global__ void __launch_bounds__(kPfThreads, kPfCtasPerSm)
    attn_shared_prefix_kernel(const __grid_constant__ CUtensorMap qmap,
                              const __grid_constant__ CUtensorMap kmap,
                              const __grid_constant__ CUtensorMap vmap, SharedPrefixArgs a) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ PrefillBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int s_err;
    constexpr bool kSplitP = Elem<T>::kDtype == KVB_BF16;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~uintptr_t(1023));
    uint8_t* sq = smem;             // Q
    uint8_t* skv = sq + kPfQBytes;  // [stage][K | V]

    asm volatile("griddepcontrol.launch_dependents;");
    const int kvh = blockIdx.x, split = blockIdx.y;
    const int seq0 = blockIdx.z * a.seqs_per_tile;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.seqs_per_tile * a.group;  // <= 128
    const int j0 = (int)((long long)split * a.n_tiles / a.splits);
    const int nt = (int)((long long)(split + 1) * a.n_tiles / a.splits) - j0;
    const int key0 = j0 * kPfKeys;

    if (tid == 0) {
        mbar_init(&bars.q_full, 1);
        for (int s = 0; s < kPfStages; ++s) {
            mbar_init(&bars.kv_full[s], 1);
            mbar_init(&bars.kv_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bars.s_full[b], 1);
            mbar_init(&bars.p_full[b], kPfRows);
        }
        mbar_init(&bars.pv_done, 1);
        mbar_init(&bars.o_done, 1);
        mbar_init(&bars.mma_done, 1);
        s_err = 0;
        fence_mbar_init();
    }
    // Rows that no sequence fills: zeros (their scores are 0 and never rescale).
    for (int i = rows * 8 + tid; i < kPfRows * 8; i += kPfThreads)
        reinterpret_cast<uint4*>(sq)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_async_smem();
    if (warp == kMmaWarp) tmem_alloc(&tmem_slot, kPfTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t fmt = Elem<T>::kDtype == KVB_BF16 ? 1u : 0u;

    if (warp == kTmaWarp) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            tma_prefetch_desc(&kmap);
            tma_prefetch_desc(&vmap);
            mbar_expect_tx(&bars.q_full, (uint32_t)(rows * 128));
            tma_load_3d(sq, &qmap, &bars.q_full, 0, kvh * a.group, seq0);
            int issued = 0;
            for (int j = 0; j < nt; ++j) {
                const int st = j % kPfStages;
                if (j >= kPfStages && !mbar_wait(&bars.kv_empty[st], ((j - kPfStages) / kPfStages) & 1)) {
                    s_err = 1;
                    break;
                }
                if (s_err) break;
                uint8_t* kdst = skv + (2 * st) * kPfKVBytes;
                uint8_t* vdst = kdst + kPfKVBytes;
                const int kt = key0 + j * kPfKeys;
                if (!a.block_table) {
                    mbar_expect_tx(&bars.kv_full[st], 2 * kPfKVBytes);
                    tma_load_3d(kdst, &kmap, &bars.kv_full[st], 0, kt, kvh);
                    tma_load_3d(vdst, &vmap, &bars.kv_full[st], 0, kt, kvh);
                } else {
                    // 32-key pieces, each inside one block; pieces past the prefix are not
                    // loaded.  An entry outside the pool is reported and reads as zeros.
                    int prow[kPfPagedPieces];
                    uint32_t bytes = 0;
#pragma unroll
                    for (int i = 0; i < kPfPagedPieces; ++i) {
                        const int k = kt + i * kPfPagedPiece;
                        prow[i] = -1;
                        if (k >= a.prefix) continue;
                        const int lb = k / a.block_size;
                        const int blk = a.block_table[lb];
                        if (blk < 0 || blk >= a.n_blocks) {
                            raise_dev_error(kDevErrBadPosition);
                            prow[i] = a.n_blocks * a.n_kv * a.block_size;
                        } else {
                            prow[i] = (blk * a.n_kv + kvh) * a.block_size + (k - lb * a.block_size);
                        }
                        bytes += 2 * kPfPagedPiece * 128;
                    }
                    mbar_expect_tx(&bars.kv_full[st], bytes);
#pragma unroll
                    for (int i = 0; i < kPfPagedPieces; ++i) {
                        if (prow[i] < 0) continue;
                        tma_load_2d(kdst + i * kPfPagedPiece * 128, &kmap, &bars.kv_full[st], 0,
                                    prow[i]);
                        tma_load_2d(vdst + i * kPfPagedPiece * 128, &vmap, &bars.kv_full[st], 0,
                                    prow[i]);
                    }
                }
                issued = j + 1;
            }
            if (s_err) {
                // let every copy this CTA issued land before the CTA exits (bounded)
                for (int j = max(0, issued - kPfStages); j < issued; ++j)
                    mbar_wait(&bars.kv_full[j % kPfStages], (j / kPfStages) & 1);
                mbar_wait(&bars.q_full, 0);
            }
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t idesc_s = idesc_f16(kPfRows, kPfKeys, fmt, 0, 0);
        const uint32_t idesc_o = idesc_f16(kPfRows, 64, fmt, 0, 1);
        const uint64_t dq = sdesc_sw128(smem_u32(sq), 16, 1024);
        const uint64_t dk0 = sdesc_sw128(smem_u32(skv), 16, 1024);
        const uint64_t dv0 = sdesc_sw128(smem_u32(skv) + kPfKVBytes, 64 * 128, 1024);
        constexpr uint64_t kStage = (2 * kPfKVBytes) >> 4;
        auto issue_s = [&](int j) {
            const uint32_t d = tmem + (uint32_t)((j & 1) * kPfKeys);
            const uint64_t db = dk0 + kStage * (j % kPfStages);
            umma_f16(d, dq, db, idesc_s, 0);
            umma_f16(d, dq + 2, db + 2, idesc_s, 1);
            umma_f16(d, dq + 4, db + 4, idesc_s, 1);
            umma_f16(d, dq + 6, db + 6, idesc_s, 1);
            umma_commit(&bars.s_full[j & 1]);
        };
        auto issue_pv = [&](int j) {
            const uint32_t d = tmem + kPfTmemO;
            const uint32_t p = tmem + (uint32_t)((j & 1) * kPfKeys);
            const uint64_t dv = dv0 + kStage * (j % kPfStages);
            umma_f16_ts(d, p, dv, idesc_o, j > 0 ? 1u : 0u);
#pragma unroll
            for (int k = 1; k < kPfKeys / 16; ++k) umma_f16_ts(d, p + 8 * k, dv + 128 * k, idesc_o, 1);
            if (kSplitP) {
#pragma unroll
                for (int k = 0; k < kPfKeys / 16; ++k)
                    umma_f16_ts(d, p + kPfPCols + 8 * k, dv + 128 * k, idesc_o, 1);
            }
            umma_commit(&bars.pv_done);
        };
        bool ok = nt > 0 && warp_all(mbar_wait(&bars.q_full, 0));
        for (int j = 0; j < 2 && j < nt && ok; ++j) {
            ok = warp_all(mbar_wait(&bars.kv_full[j % kPfStages], (j / kPfStages) & 1));
            if (ok) issue_s(j);
        }
        for (int j = 0; j < nt && ok; ++j) {
            ok = warp_all(!s_err && mbar_wait(&bars.p_full[j & 1], (j >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const int past = a.prefix - (key0 + j * kPfKeys);  // first row past the prefix
            if (a.block_table && past < kPfKeys) {
                // V rows past the prefix hold whatever the stage or the block holds there;
                // P is 0 on them, but 0 * NaN is not 0.
                uint4* vt = reinterpret_cast<uint4*>(skv + (2 * (j % kPfStages) + 1) * kPfKVBytes);
                for (int i = past * 8 + lane; i < kPfKeys * 8; i += 32)
                    vt[i] = make_uint4(0u, 0u, 0u, 0u);
                fence_async_smem();
                __syncwarp();
            }
            issue_pv(j);
            if (j + 1 == nt) umma_commit(&bars.o_done);
            if (j + 2 < nt) {
                ok = warp_all(mbar_wait(&bars.kv_full[(j + 2) % kPfStages], ((j + 2) / kPfStages) & 1));
                if (!ok) break;
                issue_s(j + 2);
            }
            umma_commit(&bars.kv_empty[j % kPfStages]);
        }
        if (!ok && nt > 0 && lane == 0) s_err = 1;
        umma_commit(&bars.mma_done);
        mbar_wait(&bars.mma_done, 0);
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax warps
        const int row = warp * 32 + lane;
        const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
        const uint32_t t_o = tmem + kPfTmemO + lane_off;
        const int seq = seq0 + row / a.group, head = row % a.group;
        const bool valid = row < rows && seq < a.n_seq;
        int limit = a.prefix;  // this row's keys
        if (a.lens && valid) limit = min(limit, max(0, min(a.lens[seq], a.max_len)));
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < nt; ++j) {
            const int b = j & 1;
            const uint32_t t_s = tmem + (uint32_t)(b * kPfKeys) + lane_off;
            ok = warp_all(!s_err && mbar_wait(&bars.s_full[b], (j >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            float s[kPfKeys];
#pragma unroll
            for (int c = 0; c < kPfKeys; c += 32) tmem_ld32(t_s + c, s + c);
            tmem_wait_ld();
            const int n_here = limit - (key0 + j * kPfKeys);
            if (n_here < kPfKeys) {
#pragma unroll
                for (int c = 0; c < kPfKeys; ++c)
                    if (c >= n_here) s[c] = -INFINITY;
            }
            float mx8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) mx8[i] = s[i];
#pragma unroll
            for (int c = 8; c + 16 <= kPfKeys; c += 16)
#pragma unroll
                for (int i = 0; i < 8; ++i) mx8[i] = max3f(mx8[i], s[c + i], s[c + 8 + i]);
            if ((kPfKeys - 8) % 16 != 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) mx8[i] = fmaxf(mx8[i], s[kPfKeys - 8 + i]);
            }
            const float mt = max3f(max3f(mx8[0], mx8[1], mx8[2]), max3f(mx8[3], mx8[4], mx8[5]),
                                   fmaxf(mx8[6], mx8[7])) *
                             a.scale_log2;
            float alpha = 1.f;
            bool rescale = false;
            if (mt > m + kPfRescaleLog2) {
                alpha = ex2_approx(m - mt);  // 0 where m is -inf
                rescale = j > 0 && m != -INFINITY;
                m = mt;
            }
            const float ref = m == -INFINITY ? 0.f : m;  // no key yet: P = 2^(-inf) = 0
            uint64_t sum2[4] = {0, 0, 0, 0};
#pragma unroll
            for (int ch = 0; ch < kPfKeys / 32; ++ch) {
                uint32_t ph[16], pl[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float p0 = ex2_approx(fmaf(s[32 * ch + 2 * k], a.scale_log2, -ref));
                    const float p1 = ex2_approx(fmaf(s[32 * ch + 2 * k + 1], a.scale_log2, -ref));
                    sum2[k & 3] = f2_add(sum2[k & 3], f2_pack(p0, p1));
                    if (kSplitP) split_bf16_pair(p0, p1, ph[k], pl[k]);
                    else ph[k] = pack_f16x2(p0, p1);
                }
                tmem_st16(t_s + 16 * ch, ph);
                if (kSplitP) tmem_st16(t_s + kPfPCols + 16 * ch, pl);
            }
            float r0, r1, r2, r3;
            f2_unpack(f2_add(sum2[0], sum2[1]), r0, r1);
            f2_unpack(f2_add(sum2[2], sum2[3]), r2, r3);
            l = l * alpha + ((r0 + r1) + (r2 + r3));
            if (__any_sync(0xffffffffu, rescale)) {
                ok = warp_all(!s_err && mbar_wait(&bars.pv_done, (j - 1) & 1));
                if (!ok) break;
                tc_fence_after();
                const float f = rescale ? alpha : 1.f;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    float o[32];
                    tmem_ld32(t_o + 32 * hf, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int d = 0; d < 32; ++d) o[d] *= f;
                    tmem_st32(t_o + 32 * hf, o);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars.p_full[b]);
        }
        if (ok && nt > 0) ok = warp_all(!s_err && mbar_wait(&bars.o_done, 0));
        if (!ok) s_err = 1;
        // The partial of this row: O, m, l.  A slice that failed contributes nothing.
        const bool have = ok && nt > 0;
        if (have) tc_fence_after();
        float* part = a.ws + (((size_t)(valid ? seq : 0) * a.n_kv + kvh) * a.max_parts + split) *
                                 (size_t)(a.group * 66);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            float o[32];
            if (have) {
                tmem_ld32(t_o + 32 * hf, o);
                tmem_wait_ld();
            } else {
#pragma unroll
                for (int d = 0; d < 32; ++d) o[d] = 0.f;
            }
            if (valid) {
                // 8-byte stores: a partial of group * 66 floats starts at any multiple of 8 bytes
                float2* dst = reinterpret_cast<float2*>(part + head * 64 + 32 * hf);
#pragma unroll
                for (int d = 0; d < 16; ++d) dst[d] = make_float2(o[2 * d], o[2 * d + 1]);
            }
        }
        if (valid) {
            part[a.group * 64 + head] = have ? m : -INFINITY;
            part[a.group * 65 + head] = have ? l : 0.f;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kPfTmemCols);
    }
}

}  // namespace kvb
