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
// A CTA takes kGroups row tiles against the same keys: 64-key K/V tiles come through a ring
// once for all of them (TMA producer warp).  Each group has four warps, one row per thread,
// which turn S (TMEM) into P (over it).  An MMA warp for every two groups issues their
// O += P V and next S = Q K^T, taking whichever group's P is ready: in a fixed order the
// groups queue for it, one warp for four groups is busy 830 cycles of every group's tile,
// and a softmax warp that issues for its own group takes ~1000 cycles a tile to do so.
// What bounds the kernel is the softmax: 16 exponentials per SM and clock (the 134 M of 1024
// rows x 8 heads x 16384 keys are 30 us; that pipe is 63 % busy) and the ~1000 cycles from a
// tile's P to its next S.  So the layout is for independent streams: a group has one S buffer
// and O, 128 TMEM columns, four groups fill an SM's 512, and the others compute while one
// waits.  The groups of a CTA stay within the ring's depth of each other; four CTAs of one
// group each do not -- the SM's schedulers favour the oldest, whose slices end early and leave
// the youngest alone (measured 41 to 71 us for equal slices).  A thread reads its scores from
// TMEM 32 at a time (maximum, then exponentials).  There is no causal mask; a row's keys end
// at the prefix's end, or for a paged sequence shorter than the prefix at its last whole 64 keys
// (the rest of them are its own kernel's).  The row's O is stored when the first tile past them
// comes: the products go on for the other rows, and 0 * V is not 0 where V holds a NaN or an
// infinity.
// Measured no better: a part of the exponentials as polynomials on the FMA pipe, halves of 32 keys
// with an S buffer each (110 us; N = 32 products cost the tensor pipe as much as N = 64).
// Measured on B200 with the own keys and the join: 256 sequences of 32 + 8 heads on 16384 keys
// with up to 1000 own, in a graph, 101 us (f16) and 107 to 114 us (bf16, P in two halves).  One row
// tile a CTA is held to 80 registers for four CTAs per SM and spills (bf16: 64 bytes a thread).
#pragma once

#include "attn_decode_q8.cuh"
#include "attn_prefill.cuh"

namespace kvb {

constexpr int kSpRows = 128, kSpKeys = 64, kSpMaxGroups = 4;
constexpr int kSpQBytes = kSpRows * 128, kSpKVBytes = kSpKeys * 128;
constexpr uint32_t kSpTmemGroup = 128, kSpTmemO = 64;  // a group's S (P over it), then O
__host__ __device__ constexpr int sp_stages(int groups) { return groups == 1 ? 2 : 3; }
__host__ __device__ constexpr int sp_smem_bytes(int groups) {
    return groups * kSpQBytes + sp_stages(groups) * 2 * kSpKVBytes + 1024;
}
// one TMA warp, and an MMA warp for every two groups
__host__ __device__ constexpr int sp_mma_warps(int groups) { return (groups + 1) / 2; }
__host__ __device__ constexpr int sp_threads(int groups) {
    return groups * 128 + 32 + 32 * sp_mma_warps(groups);
}

struct SharedBars {
    uint64_t q_full;
    uint64_t kv_full[3], kv_empty[3];
    // S of tile j (phase j), and so P V of the tile before; phase nt: O is final
    uint64_t s_full[kSpMaxGroups];
    uint64_t p_full[kSpMaxGroups];  // 128 arrivals: P of tile j is in TMEM
    uint64_t mma_done;              // every MMA of the CTA has completed
};

struct SharedPrefixArgs {
    int n_seq, n_kv, group, seqs_per_tile, row_tiles;
    int prefix;           // keys of the prefix
    int n_tiles, splits;  // 64-key tiles of the prefix, slices they are dealt to
    float scale_log2;
    const int32_t* lens;  // kShort: lengths that may end inside the prefix
    int max_len;
    float* ws;  // partials [n_seq][n_kv][max_parts][part_floats]; slice i is part i
    int max_parts, part_floats;
    const int32_t* block_table;  // row 0 holds the prefix's blocks; nullptr = contiguous
    int block_size, n_blocks;
};

// S (128 x 64, f32) = Q K^T over 64 dims: four K = 16 steps of 32 bytes along the swizzled
// 128-byte rows, then the arrival on `bar` once they are done.  One election and one block:
// an issue costs ~30 cycles then, against ~55 through umma_f16 with descriptors that move.
__device__ __forceinline__ void umma_s_64(uint32_t d, uint64_t q, uint64_t k, uint32_t idesc,
                                          uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e, p, z;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.eq.u32 p, 0, 0;\n\tsetp.ne.u32 z, 0, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, z;\n\t"
        "add.u64 a, %1, 2;\n\tadd.u64 b, %2, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.u64 a, %1, 4;\n\tadd.u64 b, %2, 4;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.u64 a, %1, 6;\n\tadd.u64 b, %2, 6;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t}" ::"r"(d),
        "l"(q), "l"(k), "r"(idesc), "r"(smem_u32(bar))
        : "memory");
}
// O += P V over 64 keys: P of keys 16 k .. in columns 32 (k / 2) + 8 (k % 2) of `p`, kSplit's
// remainders 16 columns on; V read MN-major, 16 keys (2048 bytes) per step.
template <bool kSplit>
__device__ __forceinline__ void umma_pv_64(uint32_t d, uint32_t p, uint64_t v, uint32_t idesc,
                                           uint32_t accumulate) {
    if (kSplit) {
        asm volatile(
            "{\n\t.reg .pred e, p, t;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.u32 p, %4, 0;\n\tsetp.eq.u32 t, 0, 0;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
            "add.u32 a, %1, 16;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], %2, %3, t;\n\t"
            "add.u32 a, %1, 8;\n\tadd.u64 b, %2, 128;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
            "add.u32 a, %1, 24;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
            "add.u32 a, %1, 32;\n\tadd.u64 b, %2, 256;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
            "add.u32 a, %1, 48;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
            "add.u32 a, %1, 40;\n\tadd.u64 b, %2, 384;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
            "add.u32 a, %1, 56;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t}" ::"r"(d),
            "r"(p), "l"(v), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred e, p, t;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.u32 p, %4, 0;\n\tsetp.eq.u32 t, 0, 0;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
            "add.u32 a, %1, 8;\n\tadd.u64 b, %2, 128;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
            "add.u32 a, %1, 32;\n\tadd.u64 b, %2, 256;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
            "add.u32 a, %1, 40;\n\tadd.u64 b, %2, 384;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t}" ::"r"(d),
            "r"(p), "l"(v), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}

// kShort: a.lens may end a row inside the prefix (paged).
template <typename T, int kGroups, bool kShort>
__global__ void __launch_bounds__(sp_threads(kGroups), kSpMaxGroups / kGroups)
    attn_shared_prefix_kernel(const __grid_constant__ CUtensorMap qmap,
                              const __grid_constant__ CUtensorMap kmap,
                              const __grid_constant__ CUtensorMap vmap, SharedPrefixArgs a) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ SharedBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int s_err;
    // bf16: P as head + remainder (2^-15 of a weight).  f16: one f16, P = 2^(7 + s - m) of at most
    // 2^15 (m is within 2^8 of the row's maximum): half a step, 2^-11 of a weight, or 2^-32 of 2^m
    // where it is below 2^-21 of that; a remainder would double the P V products.
    constexpr bool kSplitP = Elem<T>::kDtype == KVB_BF16;
    constexpr float kShift = kSplitP ? 0.f : 7.f;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~uintptr_t(1023));
    constexpr int kStages = sp_stages(kGroups);
    // warps: the MMA issuers, the TMA producer, the softmax warps
    constexpr int kMmas = sp_mma_warps(kGroups), kTma = kMmas, kSoftmax = kMmas + 1;
    constexpr uint32_t kTmemCols = kGroups * kSpTmemGroup;
    uint8_t* sq = smem;                       // Q of each group
    uint8_t* skv = sq + kGroups * kSpQBytes;  // [stage][K | V]

    const int kvh = blockIdx.x, split = blockIdx.y;
    const int tile0 = blockIdx.z * kGroups;  // this CTA's row tiles
    const int n_groups = min(kGroups, a.row_tiles - tile0);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.seqs_per_tile * a.group;  // <= 128
    const int j0 = (int)((long long)split * a.n_tiles / a.splits);
    const int nt = (int)((long long)(split + 1) * a.n_tiles / a.splits) - j0;  // >= 1
    const int key0 = j0 * kSpKeys;

    if (tid == 0) {
        mbar_init(&bars.q_full, 1);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&bars.kv_full[s], 1);
            mbar_init(&bars.kv_empty[s], (uint32_t)n_groups);
        }
        for (int g = 0; g < kGroups; ++g) {
            mbar_init(&bars.s_full[g], 1);
            mbar_init(&bars.p_full[g], kSpRows);
        }
        mbar_init(&bars.mma_done, kMmas);
        s_err = 0;
        fence_mbar_init();
    }
    // Rows that no sequence fills: zeros (their scores are 0 and never rescale).
    for (int g = 0; g < kGroups; ++g)
        for (int i = rows * 8 + tid; i < kSpRows * 8; i += sp_threads(kGroups))
            reinterpret_cast<uint4*>(sq + g * kSpQBytes)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_async_smem();
    // Nothing global is read or written, and no TMEM is taken, while the kernel before may run.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) tmem_alloc(&tmem_slot, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // Only now may the chain behind this grid start: its first kernel relies on everything before
    // this one, and a later one that allocates TMEM ahead of its own wait then finds every CTA of
    // this one with its columns.
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t fmt = Elem<T>::kDtype == KVB_BF16 ? 1u : 0u;

    if (warp == kTma) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            tma_prefetch_desc(&kmap);
            tma_prefetch_desc(&vmap);
            mbar_expect_tx(&bars.q_full, (uint32_t)(n_groups * rows * 128));
            for (int g = 0; g < n_groups; ++g)
                tma_load_3d(sq + g * kSpQBytes, &qmap, &bars.q_full, 0, kvh * a.group,
                            (tile0 + g) * a.seqs_per_tile);
            int issued = 0;
            for (int j = 0; j < nt; ++j) {
                const int st = j % kStages;
                if (j >= kStages && !mbar_wait(&bars.kv_empty[st], ((j - kStages) / kStages) & 1)) {
                    s_err = 1;
                    break;
                }
                if (s_err) break;
                uint8_t* kdst = skv + (2 * st) * kSpKVBytes;
                uint8_t* vdst = kdst + kSpKVBytes;
                const int kt = key0 + j * kSpKeys;
                if (!a.block_table) {
                    mbar_expect_tx(&bars.kv_full[st], 2 * kSpKVBytes);
                    tma_load_3d(kdst, &kmap, &bars.kv_full[st], 0, kt, kvh);
                    tma_load_3d(vdst, &vmap, &bars.kv_full[st], 0, kt, kvh);
                } else {
                    // The tile lies inside one block (both are multiples of 64 keys, and the
                    // prefix is whole tiles).  An entry outside the pool is reported and reads
                    // as zeros (rows past the map).
                    const int lb = kt / a.block_size;
                    const int blk = a.block_table[lb];
                    int row = a.n_blocks * a.n_kv * a.block_size;
                    if (blk < 0 || blk >= a.n_blocks) raise_dev_error(kDevErrBadPosition);
                    else row = (blk * a.n_kv + kvh) * a.block_size + (kt - lb * a.block_size);
                    mbar_expect_tx(&bars.kv_full[st], 2 * kSpKVBytes);
                    tma_load_2d(kdst, &kmap, &bars.kv_full[st], 0, row);
                    tma_load_2d(vdst, &vmap, &bars.kv_full[st], 0, row);
                }
                issued = j + 1;
            }
            if (s_err) {
                // let every copy this CTA issued land before the CTA exits (bounded)
                for (int j = max(0, issued - kStages); j < issued; ++j)
                    mbar_wait(&bars.kv_full[j % kStages], (j / kStages) & 1);
                mbar_wait(&bars.q_full, 0);
            }
        }
    } else if (warp < kMmas) {
        // ------------------------------------------------------------ MMA issuer
        // The whole warp stays converged; one elected lane issues.  Per group P_j V_j, then
        // S_{j+1} into the columns that P_j was read from: one thread's MMAs execute in order.
        const uint32_t idesc_s = idesc_f16(kSpRows, kSpKeys, fmt, 0, 0);
        const uint32_t idesc_o = idesc_f16(kSpRows, 64, fmt, 0, 1);
        const uint64_t dq0 = sdesc_sw128(smem_u32(sq), 16, 1024);
        const uint64_t dk0 = sdesc_sw128(smem_u32(skv), 16, 1024);
        const uint64_t dv0 = sdesc_sw128(smem_u32(skv) + kSpKVBytes, 64 * 128, 1024);
        constexpr uint64_t kStage = (2 * kSpKVBytes) >> 4;
        auto issue_s = [&](int g, int j) {
            umma_s_64(tmem + g * kSpTmemGroup, dq0 + (uint64_t)(g * (kSpQBytes >> 4)),
                      dk0 + kStage * (j % kStages), idesc_s, &bars.s_full[g]);
        };
        bool ok = warp_all(mbar_wait(&bars.q_full, 0) && mbar_wait(&bars.kv_full[0], 0));
        // this warp's groups: warp, warp + kMmas; next: the tile whose P is awaited
        constexpr int kMine = (kGroups + kMmas - 1) / kMmas;
        int next[kMine];
        int left = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int g = warp + i * kMmas;
            next[i] = g < n_groups ? 0 : nt;
            if (ok && g < n_groups) {
                issue_s(g, 0);
                ++left;
            }
        }
        uint64_t last = globaltimer_ns();
        int idle = 0;
        while (left > 0) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int j = next[i], g = warp + i * kMmas;
                if (j >= nt || !warp_all(mbar_test_wait(&bars.p_full[g], j & 1))) continue;
                const bool more = j + 1 < nt;
                if (more && !warp_all(mbar_test_wait(&bars.kv_full[(j + 1) % kStages],
                                                     ((j + 1) / kStages) & 1)))
                    continue;
                any = true;
                tc_fence_after();
                const uint64_t dv = dv0 + kStage * (j % kStages);
                const uint32_t t = tmem + g * kSpTmemGroup;
                umma_pv_64<kSplitP>(t + kSpTmemO, t, dv, idesc_o, j > 0 ? 1u : 0u);
                if (more) issue_s(g, j + 1);
                else umma_commit(&bars.s_full[g]);  // O is final
                umma_commit(&bars.kv_empty[j % kStages]);
                next[i] = j + 1;
                left -= more ? 0 : 1;
            }
            // a bounded wait: no group has moved for kWaitLimitNs, or another role has failed
            if (any) {
                idle = 0;
            } else if (++idle % 64 == 0) {
                const uint64_t now = globaltimer_ns();
                if (idle == 64) last = now;
                if (__any_sync(0xffffffffu, now - last > kWaitLimitNs || s_err)) {
                    if (lane == 0) raise_dev_error(kDevErrWaitTimeout);
                    ok = false;
                    break;
                }
            }
        }
        if (!ok && lane == 0) s_err = 1;
        __syncwarp();
        umma_commit(&bars.mma_done);
        mbar_wait(&bars.mma_done, 0);  // no MMA may still be running when TMEM is released
        __syncwarp();
    } else if ((warp - kSoftmax) / 4 < n_groups) {
        // ------------------------------------------------------------ softmax warps
        const int grp = (warp - kSoftmax) / 4, quarter = warp % 4;  // a warp's TMEM lanes: 32 quarter ..
        const int row = quarter * 32 + lane;
        const uint32_t t_s = tmem + grp * kSpTmemGroup + ((uint32_t)(quarter * 32) << 16);
        const uint32_t t_o = t_s + kSpTmemO;  // S, then P, at t_s
        const int seq = (tile0 + grp) * a.seqs_per_tile + row / a.group, head = row % a.group;
        const bool valid = row < rows && seq < a.n_seq;
        int limit = a.prefix;  // this row's keys
        if (kShort && valid) limit = own_key0(max(0, min(a.lens[seq], a.max_len)), limit);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        auto part_of_row = [&] {
            return (((size_t)(valid ? seq : 0) * a.n_kv + kvh) * a.max_parts + split) *
                   (size_t)a.part_floats;
        };
        for (int j = 0; j < nt; ++j) {
            ok = warp_all(!s_err && mbar_wait(&bars.s_full[grp], j & 1));
            if (!ok) break;
            tc_fence_after();
            const int n_here = limit - (key0 + j * kSpKeys);
            const bool masked = __any_sync(0xffffffffu, n_here < kSpKeys);
            float s[32];
            // The first tile past a shorter row's keys (whole tiles; where the slice begins past
            // them the part has no weight)
            if (kShort && masked && j > 0 && __any_sync(0xffffffffu, n_here == 0)) {
                float* to = a.ws + part_of_row() + head * 64;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    tmem_ld32(t_o + 32 * hf, s);
                    tmem_wait_ld();
                    if (n_here == 0)
#pragma unroll
                        for (int c = 0; c < 32; c += 4)
                            *reinterpret_cast<float4*>(to + 32 * hf + c) =
                                make_float4(s[c], s[c + 1], s[c + 2], s[c + 3]);
                }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kSpKeys; c += 32) {
                tmem_ld32(t_s + c, s);
                tmem_wait_ld();
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c + i >= n_here) s[i] = -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 32; i += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) mx[u] = max3f(mx[u], s[i + 2 * u], s[i + 2 * u + 1]);
            }
            const float mt = fmaxf(max3f(mx[0], mx[1], mx[2]), mx[3]) * a.scale_log2;
            // m is raised only past 2^8: P <= 2^(8 + kShift) then, and O and l are rescaled rarely
            float alpha = 1.f;
            bool rescale = false;
            if (mt > m + kPfRescaleLog2) {
                alpha = ex2_approx(m - mt);  // 0 where m is -inf
                rescale = m != -INFINITY;
                m = mt;
            }
            const float ref = (m == -INFINITY ? 0.f : m) - kShift;  // no key yet: P = 2^(-inf) = 0
            if (__any_sync(0xffffffffu, rescale)) {  // S(j) is there, so P(j-1) V is complete
                const float f = rescale ? alpha : 1.f;
#pragma unroll
                for (int d0 = 0; d0 < 64; d0 += 16) {
                    float o[16];
                    tmem_ld16(t_o + d0, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int d = 0; d < 16; ++d) o[d] *= f;
                    tmem_st16(t_o + d0, reinterpret_cast<const uint32_t*>(o));
                }
            }
            // P of keys 32c .. 32c + 31 goes over their own scores' columns: heads 16-bit pairs
            // in 32c .. 32c + 15, bf16 remainders after them.  The second half's scores are
            // still in registers from the maximum; the first half's are read again.
            uint64_t sum2[2] = {0, 0};
#pragma unroll
            for (int c = 1; c >= 0; --c) {
                if (c == 0) {
                    tmem_ld32(t_s, s);
                    tmem_wait_ld();
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i >= n_here) s[i] = -INFINITY;
                    }
                }
                uint32_t ph[16], pl[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float p0 = ex2_approx(fmaf(s[2 * k], a.scale_log2, -ref));
                    const float p1 = ex2_approx(fmaf(s[2 * k + 1], a.scale_log2, -ref));
                    sum2[k & 1] = f2_add(sum2[k & 1], f2_pack(p0, p1));
                    if (kSplitP) split_bf16_pair(p0, p1, ph[k], pl[k]);
                    else ph[k] = pack_f16x2(p0, p1);
                }
                tmem_st16(t_s + 32 * c, ph);
                if (kSplitP) tmem_st16(t_s + 32 * c + 16, pl);
            }
            float r0, r1;
            f2_unpack(f2_add(sum2[0], sum2[1]), r0, r1);
            l = l * alpha + (r0 + r1);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars.p_full[grp]);
        }
        if (ok) ok = warp_all(!s_err && mbar_wait(&bars.s_full[grp], nt & 1));  // O is final
        if (ok) tc_fence_after();
        else s_err = 1;
        // The partials: O, m, l of each row.  A slice that failed contributes nothing.  A
        // warp's 32 rows go through its quarter of the group's Q tile (its MMAs are done), 32
        // dims at a time, so that eight lanes store a row's 128 bytes: a thread storing its own
        // row touches 32 lines an instruction.
        const size_t off = part_of_row();
        if (valid) {
            a.ws[off + a.group * 64 + head] = ok ? m - kShift : -INFINITY;  // what O and l are relative to
            a.ws[off + a.group * 65 + head] = ok ? l : 0.f;
        }
        // else O is stored, or void
        const bool whole = valid && (!kShort || limit > key0 + (nt - 1) * kSpKeys);
        const long long dst = whole ? (long long)(off + head * 64) : -1;
        float4* stage = reinterpret_cast<float4*>(sq + grp * kSpQBytes + quarter * 4096);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            float o[32];
            if (ok) {
                tmem_ld32(t_o + 32 * hf, o);
                tmem_wait_ld();
            } else {
#pragma unroll
                for (int d = 0; d < 32; ++d) o[d] = 0.f;
            }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 8; ++c)
                stage[lane * 8 + (c ^ (lane & 7))] =
                    make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = 4 * i + lane / 8, c = lane % 8;
                const long long to = __shfl_sync(0xffffffffu, dst, r);
                if (to >= 0)
                    *reinterpret_cast<float4*>(a.ws + to + 32 * hf + 4 * c) =
                        stage[r * 8 + (c ^ (r & 7))];
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

}  // namespace kvb
