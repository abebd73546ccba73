// attention4_prompt.cuh: attention of many query rows of a sequence over the 4-bit cache (attention4.cuh), on the
// 5th-generation tensor cores: f16 and bf16 rows, where reading the cache is nothing beside the products.
//
// A CTA takes 256 query rows of a KV head as two tiles of 128 (rows token-major, the KV head's query heads side by
// side), and all positions they see, 128 at a time:
//   warps 8-14   read a tile's records and write values (8-11) and keys (12-14) as f16, f16(m + d code), into shared
//                memory (K-major, 128-byte swizzle, two stages each), 8 positions of 512 contiguous bytes of codes at a
//                time, each loaded a tile ahead. Keys [pos][dim] in the order of a lane's words (below: trx_a4p_key), the
//                queries' too; values transposed [dim][pos]: a lane's pairs of positions are the fragments that stmatrix
//                stores as rows, dim 32 g + 4 n + i in row 32 g + 8 i + n (O's columns are put right at the end)
//   warp 15      one thread issues tcgen05.mma (kind::f16, f32 accumulators in tensor memory): S = Q K^T and O += P V, the
//                tiles in turn, so that one's products run under the other's softmax
//   warps 0-7    a thread a row, 64 scores at a time: 2^(s - ref) as f16 back into tensor memory (P takes S's place) and
//                their sum, against the reference of the scores before; where one passes it by 2^8, the references of
//                the warp's rows move up and O, P and the sums so far are rescaled (p stays below 2^15)
// What bounds it: each tile's own chain, a softmax pass (2200 to 2800 cycles for 128 positions) and then its products (P V
// 1000, the next Q K^T 550, with the waits between), 4800 cycles of which the other tile's softmax covers half; converting
// the records takes 3000 of the same cycles in other warps. 2 x 2048 rows of 32 heads at the end of 4096 positions: 292 us,
// 0.43 of the measured bf16 rate; 8192 rows from the first position 696 us, 0.48. The loops are kept short: with all of them
// unrolled the warps waited for instructions (480 us). Scores in two halves of 64 positions, the first of which need not wait
// for P V: 310 us (products with N = 64 read the queries twice).
// Tensor memory: S 0, S 1, O 0, O 1, 128 columns each (O: HD).
//
// The keys' and values' rounding to f16 (2^-11 relative at most) is the choice that the 16-bit rows allow: half a step of
// f16 rows, a sixteenth of bf16's. Values past f16 (|m| + 15 d > 60000, which a cache of bf16 or f32 rows may hold) make the
// CTA start again with all keys and all values multiplied by a power of two that fits the largest of its context.
// Scores of 2^22 and more (log2) make it start again too, with each product of a score and its factor rounded as the
// maximum's is: what a fused one keeps beside the reference would let p pass f16 from 2^24 on. (Rounding them always: 309 us
// for 296.)
// A NaN among the values must not reach the rows that do not see its position, though their p is 0: it is written as 0,
// and the first position of such a group is kept; rows that see it get NaN at the end.
#pragma once
#include "attention4.cuh"
#include "prefill.cuh"

#define TRX_A4P_THREADS 512
#define TRX_A4P_ROWS 256 // query rows a CTA
#define TRX_A4P_KEYS 128 // positions a tile

template <int HD> struct TrxA4P { // dynamic shared memory (from a 1024-byte boundary)
    static constexpr int Q = 128 * HD * 2, K = TRX_A4P_KEYS * HD * 2; // one tile of queries, of keys or values
    static constexpr int SMEM = 2 * Q + 4 * K + 1024;
    static constexpr uint32_t IDESC = (1u << 4) | ((128u >> 4) << 24); // D f32, A and B f16, K-major, M = 128
};

// byte of (row, 16-byte chunk) in a K-major tile with 128-byte swizzle: 64 f16 (8 chunks) a row, `rows` rows, then the
// next 64
__device__ __forceinline__ int trx_a4p_chunk(int row, int chunk, int rows) {
    return (chunk >> 3) * (rows * 128) + (row >> 3) * 1024 + (row & 7) * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

__device__ __forceinline__ void trx_a4p_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void trx_a4p_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void trx_a4p_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(trx_smem(bar)) : "memory");
}
__device__ __forceinline__ void trx_a4p_inval(uint64_t *bar) {
    asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(trx_smem(bar)) : "memory");
}
// 32 columns of this warp's rows, in flight until the wait names them
__device__ __forceinline__ void trx_a4p_landed(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void trx_a4p_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
                 "%15, %16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                 "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
// four 8 x 8 matrices of f16 fragments to shared memory, a row of 16 bytes at each lane's address (lanes 8 i .. 8 i + 7:
// matrix i)
__device__ __forceinline__ void trx_a4p_stmatrix(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
// the 16-byte chunk of a key's or query's row that holds dims 32 g + 8 c + 0 4 1 5 2 6 3 7 (eight lanes store the chunks
// c of one g of two neighbouring rows at a time: these fall into different banks)
__device__ __forceinline__ int trx_a4p_key(int g, int c) { return (g >> 1) * 8 + 2 * c + (g & 1); }
// What the f16 tiles do not take: group ends past 60000 (hi: the largest m + 15 d, a NaN stays; lo: the smallest m)
__device__ __forceinline__ void trx_a4p_ends(uint32_t d, uint32_t m, uint32_t &hi, uint32_t &lo) {
    asm("{\n .reg .b32 t;\n fma.rn.f16x2 t, %2, %4, %3;\n max.NaN.f16x2 %0, %0, t;\n min.f16x2 %1, %1, %3;\n}"
        : "+r"(hi), "+r"(lo)
        : "r"(d), "r"(m), "r"(0x4b804b80u)); // 15
}
__device__ __forceinline__ bool trx_a4p_wide(uint32_t hi, uint32_t lo) {
    const float2 h = trx_a4_float2(hi), l = trx_a4_float2(lo);
    return h.x > 60000.0f || h.y > 60000.0f || l.x < -60000.0f || l.y < -60000.0f;
}

// Every row of the warp times its f: n columns of 32-bit floats at `to`, m columns of f16 pairs at `tp`
__device__ __noinline__ void trx_a4p_rescale(uint32_t to, int n, uint32_t tp, int m, float f) {
    const uint32_t h = trx_a4_half2(f, f);
#pragma unroll 1
    for (int i = 0; i < n; i += 16) {
        uint32_t r[16];
        trx_tmem_ld16_nw(to + i, r);
        trx_tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; k++) asm volatile("mul.rn.f32 %0, %0, %1;" : "+r"(r[k]) : "r"(__float_as_uint(f)));
        trx_a4p_st16(to + i, r);
    }
#pragma unroll 1
    for (int i = 0; i < m; i += 16) {
        uint32_t r[16];
        trx_tmem_ld16_nw(tp + i, r);
        trx_tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; k++) asm volatile("mul.rn.f16x2 %0, %0, %1;" : "+r"(r[k]) : "r"(h));
        trx_a4p_st16(tp + i, r);
    }
    trx_tmem_wait_st();
}

struct TrxA4PBars {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], p_read[2], o_full[2], done;
};

// blockIdx.x = 256 query rows (the last, whose contexts are the longest, first) x KV head, z the entry
template <int HD> __global__ void __launch_bounds__(TRX_A4P_THREADS, 1)
    trx_a4_prompt(TrxA4 a, TrxA4Batch b, TrxA4Rows io, float scale) {
    using L = TrxA4L<HD>;
    using S = TrxA4P<HD>;
    constexpr int NG = L::NG, REC = L::REC, KT = TRX_A4P_KEYS;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ __align__(8) TrxA4PBars bar;
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail, s_again, s_nan[NG], s_most[2];
    int slot, row0, rows, pos0;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kv = blockIdx.x % a.n_kv, G = a.n_head / a.n_kv;
    if (!trx_a4_entry(a, b, blockIdx.z, slot, row0, rows, pos0)) return;
    const int total = rows * G, ctas = (total + TRX_A4P_ROWS - 1) / TRX_A4P_ROWS, cta = ctas - 1 - (int)(blockIdx.x / a.n_kv);
    if (cta < 0) return;
    const uint8_t *recs = a.cache + ((int64_t)slot * a.n_kv + kv) * a.n_blocks * L::BLOCK;
    const int r0 = cta * TRX_A4P_ROWS;
    int n_tiles[2]; // tiles of positions that each tile of rows sees
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int end = min(r0 + 128 * (t + 1), total);
        n_tiles[t] = end > r0 + 128 * t ? (pos0 + (end - 1) / G) / KT + 1 : 0;
    }
    const int n_all = max(n_tiles[0], n_tiles[1]);
    const int last = pos0 + (min(r0 + TRX_A4P_ROWS, total) - 1) / G; // the last position of the CTA's rows
    uint8_t *smem = smem_raw + ((1024 - (trx_smem(smem_raw) & 1023)) & 1023);
    uint8_t *sq = smem, *sk = smem + 2 * S::Q, *sv = sk + 2 * S::K;

    // ---- the queries, a thread a row
    const int t_mine = warp >> 2; // warps 0-7: the tile of rows
    int lim = -1;
    float c0 = 0.0f;
    int64_t out_at = 0;
    if (warp < 8) {
        const int r = r0 + tid, row = tid & 127;
        const bool on = r < total;
        const int tok = on ? r / G : 0;
        const int64_t head = (int64_t)(kv * G + (on ? r - tok * G : 0)) * HD;
        const int64_t at = (int64_t)(row0 + tok) * io.q_stride + head;
        out_at = (int64_t)(row0 + tok) * io.out_stride + head;
        if (on) lim = pos0 + tok;
        uint4 raw[HD / 8];
        float most = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < HD / 8; i++) {
            raw[i] = on ? reinterpret_cast<const uint4 *>((const uint16_t *)io.q + at)[i] : make_uint4(0, 0, 0, 0);
            const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = io.bf16 ? make_float2(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xffff0000u))
                                         : trx_a4_float2(u[j]);
                most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
                bad |= !(fabsf(f.x) <= 3.402823466e38f) || !(fabsf(f.y) <= 3.402823466e38f);
            }
        }
        int ex = 0;
        if (!bad && most > 0.0f) ex = max((int)((__float_as_uint(most) >> 23) & 255) - 126, -100);
        const float f = __int_as_float((10 - ex + 127) << 23) * (scale < 0.0f ? -1.0f : 1.0f);
        // (kept above 0 and in range: a masked score, -inf, stays one and a score of 0 stays 0)
        c0 = bad || !(fabsf(scale) <= 3.402823466e38f)
                 ? __int_as_float(0x7fffffff)
                 : fminf(1.0e-30f + fabsf(scale) * (1.44269504088896341f * __int_as_float((ex - 10 + 127) << 23)), 3.0e36f);
#pragma unroll
        for (int i = 0; i < HD / 8; i++) { // (dims 32 g + 8 c ..: chunk 4 g + c)
            const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            float x[8];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 y = io.bf16 ? make_float2(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xffff0000u))
                                         : trx_a4_float2(u[j]);
                x[2 * j] = bad ? 0.0f : y.x * f, x[2 * j + 1] = bad ? 0.0f : y.y * f;
            }
            *reinterpret_cast<uint4 *>(sq + t_mine * S::Q + trx_a4p_chunk(row, trx_a4p_key(i >> 2, i & 3), 128)) =
                make_uint4(trx_a4_half2(x[0], x[4]), trx_a4_half2(x[1], x[5]), trx_a4_half2(x[2], x[6]), trx_a4_half2(x[3], x[7]));
        }
        trx_fence_proxy_async();
    }
    if (warp == 15) {
        trx_tmem_alloc(&s_tmem, 512);
        trx_tmem_relinquish();
    }
    if (tid == 0) s_fail = 0, s_again = 0, s_most[0] = s_most[1] = 0;
    if (tid < NG) s_nan[tid] = INT_MAX;

    float l = 0.0f;
    int ek = 0, ev = 0; // keys and values are held times 2^-ek, 2^-ev
    for (int attempt = 0;; attempt++) {
        if (tid == 0) {
            for (int i = 0; i < 2; i++) {
                if (attempt) {
                    trx_a4p_inval(&bar.k_full[i]), trx_a4p_inval(&bar.k_empty[i]), trx_a4p_inval(&bar.v_full[i]);
                    trx_a4p_inval(&bar.v_empty[i]), trx_a4p_inval(&bar.s_full[i]), trx_a4p_inval(&bar.p_ready[i]);
                    trx_a4p_inval(&bar.o_full[i]), trx_a4p_inval(&bar.p_read[i]);
                    if (i == 0) trx_a4p_inval(&bar.done);
                }
                trx_mbar_init(&bar.k_full[i], 3), trx_mbar_init(&bar.v_full[i], 4), trx_mbar_init(&bar.p_ready[i], 4);
                trx_mbar_init(&bar.k_empty[i], 1), trx_mbar_init(&bar.v_empty[i], 1), trx_mbar_init(&bar.s_full[i], 1);
                trx_mbar_init(&bar.o_full[i], 1), trx_mbar_init(&bar.p_read[i], 1);
                if (i == 0) trx_mbar_init(&bar.done, 1);
            }
            trx_fence_barrier_init();
        }
        trx_tc_fence_before();
        __syncthreads();
        trx_tc_fence_after();
        const uint32_t tmem = s_tmem;
        auto wait = [&](uint64_t *w, int phase) {
            if (trx_mbar_wait(w, phase & 1, TRX_WAIT_NS)) return true;
            *(volatile int *)&s_fail = 1;
            return false;
        };

        if (warp < 8) {
            // ---- softmax
            const int n = n_tiles[t_mine];
            const uint32_t ts = tmem + ((uint32_t)(warp & 3) << 21) + 128 * t_mine, to = ts + 256;
            const float f = c0 * __int_as_float((ek + 127) << 23), c = f > 3.0e38f ? 3.0e38f : f; // (a NaN stays)
            constexpr float NONE = -3.0e38f; // no position seen
            float top = NONE, ref = NONE;
            trx_f2 sum = 0;
            const int low = __reduce_min_sync(0xffffffffu, lim);
            // FAR: the products s c are rounded, as the maximum's is, before the reference is subtracted
            auto tiles = [&](auto far) {
                constexpr bool FAR = decltype(far)::value;
                for (int j = 0; j < n; j++) {
                    if (!__all_sync(0xffffffffu, wait(&bar.s_full[t_mine], j))) break;
                    trx_tc_fence_after();
                    const bool mask = j * KT + KT - 1 > low;
                    const int see = lim - j * KT; // the tile's last column that the row sees
                    // 32 columns from `at`: their maximum, and p
                    auto look = [&](uint32_t(&r)[32], int at) {
                        if (mask) {
#pragma unroll
                            for (int i = 0; i < 32; i++) // (volatile: a branch, not 32 selections for every tile)
                                asm volatile("{\n .reg .pred q;\n setp.gt.s32 q, %1, %2;\n @q mov.b32 %0, 0xff800000;\n}"
                                             : "+r"(r[i])
                                             : "r"(at + i), "r"(see));
                        }
                        float best[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            best[k] = fmaxf(__uint_as_float(r[8 * k]), __uint_as_float(r[8 * k + 1]));
#pragma unroll
                            for (int i = 2; i < 8; i += 2)
                                best[k] = trx_a4_max3(best[k], __uint_as_float(r[8 * k + i]), __uint_as_float(r[8 * k + i + 1]));
                        }
                        return trx_a4_max3(fmaxf(best[0], best[1]), best[2], best[3]) * c;
                    };
                    auto take = [&](uint32_t(&r)[32], int at) {
                        uint32_t p[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            trx_f2 e = (trx_f2)r[i] | (trx_f2)r[i + 1] << 32;
                            if constexpr (FAR) e = trx_sub2(trx_mul2(e, trx_pack2(c, c)), trx_pack2(ref, ref));
                            else e = trx_fma2(e, trx_pack2(c, c), trx_pack2(-ref, -ref));
                            const float x = trx_a4_exp2(trx_lo(e)), y = trx_a4_exp2(trx_hi(e));
                            p[i / 2] = trx_a4_half2(x, y);
                            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum) : "l"(trx_pack2(x, y)));
                        }
                        trx_a4p_st16(ts + at / 2, p);
                    };
#pragma unroll 1
                    for (int h = 0; h < 128; h += 64) {
                        uint32_t r0[32], r1[32];
                        trx_tmem_ld32_nw(ts + h, r0);
                        trx_tmem_ld32_nw(ts + h + 32, r1);
                        trx_a4p_landed(r0);
                        trx_a4p_landed(r1);
                        const float best = fmaxf(look(r0, h), look(r1, h + 32));
                        if (__any_sync(0xffffffffu, best > __fadd_rd(top, 8.0f))) { // (S j is complete: so are O's products before it)
                            top = fmaxf(top, best);
                            // (rounded up, and 8 more rounded down: p must not pass f16 where scores are large)
                            const float next = top == NONE ? NONE : __fadd_ru(top, -7.0f), f = ref == next ? 1.0f : trx_a4_exp2(ref - next);
                            if (!FAR && fabsf(top) >= 4194304.0f && top != NONE) *(volatile int *)&s_again = 1;
                            ref = next;
                            sum = trx_mul2(sum, trx_pack2(f, f));
                            trx_a4p_rescale(to, j > 0 ? HD : 0, ts, h / 2, f);
                        }
                        take(r0, h);
                        take(r1, h + 32); // (S's columns h / 2 .. h / 2 + 31 have been read)
                    }
                    trx_tmem_wait_st();
                    trx_tc_fence_before();
                    __syncwarp();
                    if (lane == 0) trx_a4p_arrive(&bar.p_ready[t_mine]);
                }
            };
            if (attempt == 0) tiles(std::false_type{});
            else tiles(std::true_type{});
            l = trx_lo(sum) + trx_hi(sum);
            if (n > 0) __all_sync(0xffffffffu, wait(&bar.o_full[t_mine], 0));
            trx_tc_fence_after();
        } else if (warp < 12) {
            // ---- values to f16: 16 times 8 positions, four a warp; lane (n, c): positions 2 c, 2 c + 1, dims 32 g + 4 n ..
            struct Piece {
                uint32_t w[NG], d[NG], m[NG];
            } first, second;
            const __half2 fv = __half2half2(__ushort_as_half((uint16_t)((15 - ev) << 10)));
            const uint32_t hv = *reinterpret_cast<const uint32_t *>(&fv);
            const int cc = lane & 3, t0 = warp - 8; // 8 positions t0 + 4 q: the q-th record's t0-th
            auto load = [&](Piece &x, int pos) {
                const uint8_t *rec = recs + (int64_t)(pos >> 5) * REC;
                if (pos <= last) {
                    trx_a4_lds<NG>(rec + L::V + t0 * (4 * HD) + lane * (NG * 4), x.w);
                    trx_a4_lds<NG>(rec + L::VD + (4 * t0 + cc) * (NG * 4), x.d);
                    trx_a4_lds<NG>(rec + L::VM + (4 * t0 + cc) * (NG * 4), x.m);
                } else
#pragma unroll
                    for (int g = 0; g < NG; g++) x.w[g] = x.d[g] = x.m[g] = 0;
            };
            // stmatrix: lane 8 i + n stores the row of dim 32 g + 4 n + i
            const uint32_t rows = trx_smem(sv) + (lane >> 3) * 1024 + (lane & 7) * 128;
            auto convert = [&](Piece &x, int pos, int st, int t8) {
                if (pos + 7 > last) { // (the record's later positions)
                    const int at = pos + 2 * cc;
                    const uint32_t on = (at <= last ? 0xffffu : 0u) | (at + 1 <= last ? 0xffff0000u : 0u);
#pragma unroll
                    for (int g = 0; g < NG; g++) x.d[g] &= on, x.m[g] &= on;
                }
                uint32_t hi = 0, lo = 0;
#pragma unroll
                for (int g = 0; g < NG; g++) trx_a4p_ends(x.d[g], x.m[g], hi, lo);
                const float2 top = trx_a4_float2(hi);
                if (top.x != top.x || top.y != top.y) { // a NaN: kept apart, and 0 here (its codes and minimum are 0)
                    hi = 0;
#pragma unroll
                    for (int g = 0; g < NG; g++) {
#pragma unroll
                        for (int o = 0; o < 2; o++) // (scales are not negative: a NaN's bits are above an infinity's)
                            if (((x.d[g] >> (16 * o)) & 0xffffu) > 0x7c00u) {
                                atomicMin(&s_nan[g], pos + 2 * cc + o);
                                x.d[g] &= o ? 0xffffu : 0xffff0000u;
                            }
                        trx_a4p_ends(x.d[g], x.m[g], hi, lo);
                    }
                }
                if (trx_a4p_wide(hi, lo)) *(volatile int *)&s_again = 1;
                const uint32_t to = rows + st * S::K + (t8 >> 3) * (HD * 128) + (((t8 & 7) ^ (lane & 7)) << 4);
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    uint32_t h[4];
                    trx_a4_codes<true>(x.w[g], h);
                    if (ev) x.d[g] = trx_a4_hmul2(x.d[g], hv), x.m[g] = trx_a4_hmul2(x.m[g], hv);
                    trx_a4p_stmatrix(to + g * 4096, trx_a4_hfma2(h[0], x.d[g], x.m[g]), trx_a4_hfma2(h[1], x.d[g], x.m[g]),
                                     trx_a4_hfma2(h[2], x.d[g], x.m[g]), trx_a4_hfma2(h[3], x.d[g], x.m[g]));
                }
            };
            load(first, 8 * t0);
            load(second, 32 + 8 * t0);
#pragma unroll 1
            for (int j = 0, q = 0; j < n_all;) { // 8 positions, and the 8 a record on
                if (q == 0 && j >= 2 && !__all_sync(0xffffffffu, wait(&bar.v_empty[j & 1], (j >> 1) - 1))) break;
                const int pos = j * KT + 32 * q + 8 * t0;
                convert(first, pos, j & 1, 4 * q + t0);
                load(first, pos + 64);
                convert(second, pos + 32, j & 1, 4 * q + 4 + t0);
                load(second, pos + 96);
                if ((q += 2) == 4) {
                    trx_fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) trx_a4p_arrive(&bar.v_full[j & 1]);
                    q = 0, j++;
                }
            }
        } else if (warp < 15) {
            // ---- keys to f16: 16 times 8 positions over three warps; lane (n, c): position n, dims 32 g + 8 c ..
            struct Piece {
                uint32_t w[NG], d[NG / 2], m[NG / 2];
            } first, second;
            const __half2 fk = __half2half2(__ushort_as_half((uint16_t)((15 - ek) << 10)));
            const uint32_t hk = *reinterpret_cast<const uint32_t *>(&fk);
            const int n = lane >> 2, cc = lane & 3, x0 = warp - 12;
            auto load = [&](Piece &x, int pos) {
                const uint8_t *rec = recs + (int64_t)(pos >> 5) * REC;
                if (pos <= last) {
                    trx_a4_lds<NG>(rec + (pos & 31) * (HD / 2) + cc * (NG * 4), x.w);
                    trx_a4_lds<NG / 2>(rec + L::KD + (pos & 31) * (NG * 2), x.d);
                    trx_a4_lds<NG / 2>(rec + L::KM + (pos & 31) * (NG * 2), x.m);
                } else
#pragma unroll
                    for (int g = 0; g < NG; g++) x.w[g] = x.d[g / 2] = x.m[g / 2] = 0;
            };
            auto convert = [&](Piece &x, int st, int p) {
                uint32_t hi = 0, lo = 0;
#pragma unroll
                for (int i = 0; i < NG / 2; i++) {
                    trx_a4p_ends(x.d[i], x.m[i], hi, lo); // (beside a NaN: its scores are NaN)
                    if (ek) x.d[i] = trx_a4_hmul2(x.d[i], hk), x.m[i] = trx_a4_hmul2(x.m[i], hk);
                }
                if (trx_a4p_wide(hi, lo)) *(volatile int *)&s_again = 1;
                uint8_t *to = sk + st * S::K;
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const uint32_t half = g & 1 ? 0x3232 : 0x1010;
                    const uint32_t d = __byte_perm(x.d[g / 2], 0, half), m = __byte_perm(x.m[g / 2], 0, half);
                    uint32_t h[4];
                    trx_a4_codes<true>(x.w[g], h);
                    *reinterpret_cast<uint4 *>(to + trx_a4p_chunk(p, trx_a4p_key(g, cc), KT)) =
                        make_uint4(trx_a4_hfma2(h[0], d, m), trx_a4_hfma2(h[1], d, m), trx_a4_hfma2(h[2], d, m), trx_a4_hfma2(h[3], d, m));
                }
            };
            load(first, 8 * x0 + n);
            load(second, 8 * (x0 + 3) + n);
#pragma unroll 1
            for (int j = 0, q = 0; j < n_all;) { // (the last of six is there for warp 12 only)
                if (q == 0 && j >= 2 && !__all_sync(0xffffffffu, wait(&bar.k_empty[j & 1], (j >> 1) - 1))) break;
                const int p = 8 * (x0 + 3 * q) + n, next = q < 4 ? j * KT + p + 48 : (j + 1) * KT + 8 * x0 + n;
                convert(first, j & 1, p);
                load(first, next);
                if (p + 24 < KT) convert(second, j & 1, p + 24);
                load(second, next + 24);
                if ((q += 2) == 6) {
                    trx_fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) trx_a4p_arrive(&bar.k_full[j & 1]);
                    q = 0, j++;
                }
            }
        } else if (lane == 0) {
            // ---- products: O t += P t V of the tile before, then S t = Q t K
            const uint32_t aq = trx_smem(sq), ak = trx_smem(sk), av = trx_smem(sv);
            constexpr uint32_t is = S::IDESC | ((uint32_t)(KT >> 3) << 17), iv = S::IDESC | ((uint32_t)(HD >> 3) << 17);
            const uint64_t dq = trx_umma_desc_sw128(aq), dk = trx_umma_desc_sw128(ak), dv = trx_umma_desc_sw128(av);
            const int n0 = n_tiles[0], n1 = n_tiles[1];
            auto pv = [&](int t, int n, int j) { // O t += P t V of the tile before
                if (j == 0 || j > n) return true;
                const int st = (j - 1) & 1;
                if (!wait(&bar.p_ready[t], j - 1) || !wait(&bar.v_full[st], (j - 1) >> 1)) return false;
                trx_tc_fence_after();
                const uint64_t d = dv + (uint64_t)(st * (S::K >> 4));
#pragma unroll
                for (int k = 0; k < KT / 16; k++)
                    trx_a4p_mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k, d + (uint64_t)((k >> 2) * (HD * 8) + 2 * (k & 3)), iv,
                                   j > 1 || k > 0);
                if (j == n) trx_umma_commit(&bar.o_full[t]);
                else trx_umma_commit(&bar.p_read[t]);
                return true;
            };
            auto qk = [&](int t, int n, int j) { // S t = Q t K
                if (j >= n) return true;
                const int st = j & 1;
                // (S takes P's place: the products that read P are waited for)
                if (!wait(&bar.k_full[st], j >> 1) || (j > 0 && !wait(&bar.p_read[t], j - 1))) return false;
                trx_tc_fence_after();
                const uint64_t da = dq + (uint64_t)(t * (S::Q >> 4)), db = dk + (uint64_t)(st * (S::K >> 4));
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint64_t o = (uint64_t)((k >> 2) * (128 * 8) + 2 * (k & 3));
                    trx_a4p_mma(tmem + 128 * t, da + o, db + o, is, k > 0);
                }
                trx_umma_commit(&bar.s_full[t]);
                return true;
            };
#pragma unroll 1
            for (int j = 0; j <= n_all; j++) {
                if (!pv(0, n0, j) || !qk(0, n0, j) || !pv(1, n1, j)) break;
                if (j > 0) trx_umma_commit(&bar.v_empty[(j - 1) & 1]);
                if (!qk(1, n1, j)) break;
                if (j < n_all) trx_umma_commit(&bar.k_empty[j & 1]);
            }
            trx_umma_commit(&bar.done); // no product is in flight when the tensor memory goes
            wait(&bar.done, 0);
        }
        __syncwarp();
        trx_tc_fence_before();
        __syncthreads();
        trx_tc_fence_after();
        if (attempt > 0 || *(volatile int *)&s_again == 0 || *(volatile int *)&s_fail != 0) break;
        // the largest |m| + 15 d of the keys and of the values
        float most[2] = {0.0f, 0.0f};
        const int words = 16 * NG; // of a plane
        for (int64_t i = tid; i < (int64_t)(last / 32 + 1) * words; i += TRX_A4P_THREADS) {
            const uint8_t *rec = recs + i / words * REC + i % words * 4;
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const float2 d = trx_a4_float2(*reinterpret_cast<const uint32_t *>(rec + (x ? L::VD : L::KD)));
                const float2 m = trx_a4_float2(*reinterpret_cast<const uint32_t *>(rec + (x ? L::VM : L::KM)));
                most[x] = fmaxf(most[x], fmaxf(__fmaf_rn(d.x, 15.0f, fabsf(m.x)), __fmaf_rn(d.y, 15.0f, fabsf(m.y))));
            }
        }
        for (int x = 0; x < 2; x++) atomicMax(&s_most[x], __float_as_int(most[x]));
        __syncthreads();
        ek = max(0, ((s_most[0] >> 23) & 255) - 126 - 15), ev = max(0, ((s_most[1] >> 23) & 255) - 126 - 15);
    }
    if (warp < 8) {
        const uint32_t to = s_tmem + ((uint32_t)(warp & 3) << 21) + 256 + 128 * t_mine;
        const float f = __fdiv_rn(__int_as_float((ev + 127) << 23), l);
#pragma unroll 1
        for (int g = 0; g < NG; g++) {
            float o[32];
            __syncwarp();
            trx_tmem_ld32(to + 32 * g, o);
            if (lim < 0 || *(volatile int *)&s_fail != 0) continue;
            const float x = lim >= s_nan[g] ? __int_as_float(0x7fffffff) : f;
#pragma unroll
            for (int i = 0; i < 8; i++)
                trx_a4_out4<false>(io, out_at + 32 * g + 4 * i, make_float4(o[i] * x, o[8 + i] * x, o[16 + i] * x, o[24 + i] * x));
        }
        if (tid == 0 && s_fail) atomicCAS(a.err, 0, TRX_A4_GAVE_UP);
    }
    trx_tc_fence_before();
    __syncthreads();
    if (warp == 15) {
        trx_tc_fence_after();
        trx_tmem_dealloc(s_tmem, 512);
    }
}
