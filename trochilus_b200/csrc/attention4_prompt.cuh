// attention4_prompt.cuh: attention of many query rows of a sequence over the 4-bit cache (attention4.cuh), on the
// 5th-generation tensor cores: f16 and bf16 rows, where reading the cache is nothing beside the products.
//
// A CTA takes 256 query rows of a KV head as two tiles of 128 (rows token-major, the KV head's query heads side by
// side), and all positions they see, 128 at a time:
//   warps 8-11   read a tile's records and write keys and values as f16, f16(m + d code), into shared memory (K-major,
//                128-byte swizzle, two stages each): keys [pos][dim], in a record's word order (dims 0 4 1 5 2 6 3 7 of
//                each 8, the queries' too), values transposed [dim][pos] (a record's words hold position pairs)
//   warp 12      one thread issues tcgen05.mma (kind::f16, f32 accumulators in tensor memory): S = Q K^T and O += P V, the
//                tiles in turn, so that one's products run under the other's softmax
//   warps 0-7    a thread a row: the maximum, 2^(s - ref) as f16 back into tensor memory (P takes S's place), the sum. O
//                is rescaled only when a row's maximum passes its reference by 2^8 (p stays below 2^15).
// Tensor memory: S 0, S 1, O 0, O 1, 128 columns each (O: HD).
//
// The keys' and values' rounding to f16 (2^-12 relative) is the choice that the 16-bit rows allow: half a step of f16
// rows, a sixteenth of bf16's. Values past f16 (|m| + 15 d > 60000, which a cache of bf16 or f32 rows may hold) make the
// CTA start again with all keys and all values multiplied by a power of two that fits the largest of its context.
// A NaN among the values must not reach the rows that do not see its position, though their p is 0: it is written as 0,
// and the first position of such a group is kept; rows that see it get NaN at the end.
#pragma once
#include "attention4.cuh"
#include "prefill.cuh"

#define TRX_A4P_THREADS 416
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
__device__ __forceinline__ void trx_a4p_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
                 "%15, %16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                 "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void trx_a4p_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(trx_smem(bar)) : "memory");
}
__device__ __forceinline__ void trx_a4p_inval(uint64_t *bar) {
    asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(trx_smem(bar)) : "memory");
}
// a scale's or minimum's |m| + 15 d past what the f16 tiles take (false where d is NaN)
__device__ __forceinline__ bool trx_a4p_wide(uint32_t d, uint32_t m) {
    const float2 x = trx_a4_float2(d), y = trx_a4_float2(m);
    return fmaxf(__fmaf_rn(x.x, 15.0f, fabsf(y.x)), __fmaf_rn(x.y, 15.0f, fabsf(y.y))) > 60000.0f;
}

struct TrxA4PBars {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], o_full[2], done;
};

template <int HD> __global__ void __launch_bounds__(TRX_A4P_THREADS, 1)
    trx_a4_prompt(TrxA4 a, TrxA4Batch b, TrxA4Rows io, float scale) {
    using L = TrxA4L<HD>;
    using S = TrxA4P<HD>;
    constexpr int NG = L::NG, REC = L::REC, KT = TRX_A4P_KEYS;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ __align__(8) TrxA4PBars bar;
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail, s_wide, s_nan[NG], s_most[2];
    int slot, row0, rows, pos0;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kv = blockIdx.y, G = a.n_head / a.n_kv;
    if (!trx_a4_entry(a, b, blockIdx.z, slot, row0, rows, pos0)) return;
    const int total = rows * G, ctas = (total + TRX_A4P_ROWS - 1) / TRX_A4P_ROWS, cta = ctas - 1 - (int)blockIdx.x;
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
        c0 = bad ? __int_as_float(0x7fffffff)
                 : fminf(fabsf(scale) * 1.44269504088896341f * __int_as_float((min(ex, 120) - 10 + 127) << 23), 3.0e36f);
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
            *reinterpret_cast<uint4 *>(sq + t_mine * S::Q + trx_a4p_chunk(row, i, 128)) =
                make_uint4(trx_a4_half2(x[0], x[4]), trx_a4_half2(x[1], x[5]), trx_a4_half2(x[2], x[6]), trx_a4_half2(x[3], x[7]));
        }
        trx_fence_proxy_async();
    }
    if (warp == 12) {
        trx_tmem_alloc(&s_tmem, 512);
        trx_tmem_relinquish();
    }
    if (tid == 0) s_fail = 0, s_wide = 0, s_most[0] = s_most[1] = 0;
    if (tid < NG) s_nan[tid] = INT_MAX;

    float l = 0.0f;
    int ek = 0, ev = 0; // keys and values are held times 2^-ek, 2^-ev
    for (int attempt = 0;; attempt++) {
        if (tid == 0) {
            for (int i = 0; i < 2; i++) {
                if (attempt) {
                    trx_a4p_inval(&bar.k_full[i]), trx_a4p_inval(&bar.k_empty[i]), trx_a4p_inval(&bar.v_full[i]);
                    trx_a4p_inval(&bar.v_empty[i]), trx_a4p_inval(&bar.s_full[i]), trx_a4p_inval(&bar.p_ready[i]);
                    trx_a4p_inval(&bar.o_full[i]);
                    if (i == 0) trx_a4p_inval(&bar.done);
                }
                trx_mbar_init(&bar.k_full[i], 4), trx_mbar_init(&bar.v_full[i], 4), trx_mbar_init(&bar.p_ready[i], 4);
                trx_mbar_init(&bar.k_empty[i], 1), trx_mbar_init(&bar.v_empty[i], 1), trx_mbar_init(&bar.s_full[i], 1);
                trx_mbar_init(&bar.o_full[i], 1);
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
            const float c = fminf(c0 * __int_as_float((ek + 127) << 23), 3.0e38f);
            float top = -1.0e30f, ref = -1.0e30f;
            l = 0.0f;
            const int low = __reduce_min_sync(0xffffffffu, lim);
            for (int j = 0; j < n; j++) {
                if (!__all_sync(0xffffffffu, wait(&bar.s_full[t_mine], j))) break;
                trx_tc_fence_after();
                const bool mask = j * KT + KT - 1 > low;
                const int see = lim - j * KT; // the tile's last column that the row sees
                float s[32], best = -INFINITY;
#pragma unroll 1
                for (int h = 0; h < 4; h++) {
                    trx_tmem_ld32(ts + 32 * h, s);
                    if (mask) {
#pragma unroll
                        for (int i = 0; i < 32; i++) s[i] = 32 * h + i > see ? -INFINITY : s[i];
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 2) best = trx_a4_max3(best, s[i], s[i + 1]);
                }
                best *= c;
                if (__any_sync(0xffffffffu, best > top + 8.0f)) { // (S j is complete, so O's products before it are)
                    top = fmaxf(top, best);
                    const float next = top == -1.0e30f ? -1.0e30f : top - 7.0f, f = ref == next ? 1.0f : trx_a4_exp2(ref - next);
                    ref = next;
                    l *= f;
                    if (j > 0) {
#pragma unroll 1
                        for (int h = 0; h < HD / 32; h++) {
                            trx_tmem_ld32(to + 32 * h, s);
#pragma unroll
                            for (int i = 0; i < 32; i++) s[i] *= f;
                            trx_tmem_st32(to + 32 * h, s);
                        }
                        trx_tmem_wait_st();
                    }
                }
                trx_f2 sum = 0;
#pragma unroll 1
                for (int h = 0; h < 4; h++) {
                    trx_tmem_ld32(ts + 32 * h, s);
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float x = trx_a4_exp2(__fmaf_rn(s[i], c, -ref)), y = trx_a4_exp2(__fmaf_rn(s[i + 1], c, -ref));
                        if (mask) {
                            if (32 * h + i > see) x = 0.0f;
                            if (32 * h + i + 1 > see) y = 0.0f;
                        }
                        p[i / 2] = trx_a4_half2(x, y);
                        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum) : "l"(trx_pack2(x, y)));
                    }
                    trx_a4p_st16(ts + 16 * h, p); // (S's columns 16 h .. have been read)
                }
                l += trx_lo(sum) + trx_hi(sum);
                trx_tmem_wait_st();
                trx_tc_fence_before();
                __syncwarp();
                if (lane == 0) trx_a4p_arrive(&bar.p_ready[t_mine]);
            }
            if (n > 0) __all_sync(0xffffffffu, wait(&bar.o_full[t_mine], 0));
            trx_tc_fence_after();
        } else if (warp < 12) {
            // ---- keys and values to f16
            const int p = tid - 256;                                          // the key of a tile
            const int t8 = (lane & 7) + 8 * (warp & 1), vn = (lane >> 3) + 4 * ((warp - 8) >> 1); // 8 positions, dims 32 g + 4 vn ..
            const __half2 fk = __half2half2(__ushort_as_half((uint16_t)((15 - ek) << 10)));
            const __half2 fv = __half2half2(__ushort_as_half((uint16_t)((15 - ev) << 10)));
            const uint32_t hk = *reinterpret_cast<const uint32_t *>(&fk), hv = *reinterpret_cast<const uint32_t *>(&fv);
            bool go = true;
            for (int j = 0; j < n_all && go; j++) {
                const int st = j & 1;
                {
                    const int pos = j * KT + p;
                    const uint8_t *rec = recs + (int64_t)(pos >> 5) * REC;
                    uint32_t w[4][NG], d[NG / 2], m[NG / 2];
#pragma unroll
                    for (int i = 0; i < NG / 2; i++) d[i] = m[i] = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int g = 0; g < NG; g++) w[i][g] = 0;
                    if (pos <= last) {
#pragma unroll
                        for (int i = 0; i < 4; i++) trx_a4_lds<NG>(rec + (pos & 31) * (HD / 2) + i * (NG * 4), w[i]);
                        trx_a4_lds<NG / 2>(rec + L::KD + (pos & 31) * (NG * 2), d);
                        trx_a4_lds<NG / 2>(rec + L::KM + (pos & 31) * (NG * 2), m);
                    }
                    bool wide = false;
#pragma unroll
                    for (int i = 0; i < NG / 2; i++) {
                        wide |= trx_a4p_wide(d[i], m[i]);
                        d[i] = trx_a4_hmul2(d[i], hk), m[i] = trx_a4_hmul2(m[i], hk);
                    }
                    if (wide) *(volatile int *)&s_wide = 1;
                    if (j >= 2) go = __all_sync(0xffffffffu, wait(&bar.k_empty[st], (j >> 1) - 1));
                    if (!go) break;
                    uint8_t *to = sk + st * S::K;
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        const uint32_t dd = __byte_perm(d[g / 2], 0, g & 1 ? 0x3232 : 0x1010), mm = __byte_perm(m[g / 2], 0, g & 1 ? 0x3232 : 0x1010);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            uint32_t h[4];
                            trx_a4_codes<true>(w[i][g], h);
                            *reinterpret_cast<uint4 *>(to + trx_a4p_chunk(p, 4 * g + i, KT)) =
                                make_uint4(trx_a4_hfma2(h[0], dd, mm), trx_a4_hfma2(h[1], dd, mm), trx_a4_hfma2(h[2], dd, mm),
                                           trx_a4_hfma2(h[3], dd, mm));
                        }
                    }
                    trx_fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) trx_a4p_arrive(&bar.k_full[st]);
                }
                {
                    const int pos = j * KT + 8 * t8;
                    const uint8_t *rec = recs + (int64_t)(pos >> 5) * REC;
                    const int t = (pos & 31) >> 3;
                    uint32_t w[4][NG], d[4][NG], m[4][NG];
                    bool wide = false, nan = false;
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int g = 0; g < NG; g++) w[i][g] = d[i][g] = m[i][g] = 0;
                    if (pos <= last) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            trx_a4_lds<NG>(rec + L::V + t * (4 * HD) + (4 * vn + i) * (NG * 4), w[i]);
                            trx_a4_lds<NG>(rec + L::VD + (4 * t + i) * (NG * 4), d[i]);
                            trx_a4_lds<NG>(rec + L::VM + (4 * t + i) * (NG * 4), m[i]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) // (scales are not negative: a NaN's bits are above an infinity's)
#pragma unroll
                        for (int g = 0; g < NG; g++) nan |= (d[i][g] & 0xffffu) > 0x7c00u || (d[i][g] >> 16) > 0x7c00u;
                    if (pos + 7 > last || nan) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int g = 0; g < NG; g++)
#pragma unroll
                                for (int o = 0; o < 2; o++) {
                                    const int at = pos + 2 * i + o;
                                    const bool bad = ((d[i][g] >> (16 * o)) & 0xffffu) > 0x7c00u;
                                    if (at <= last && bad) atomicMin(&s_nan[g], at);
                                    if (at > last || bad) d[i][g] &= o ? 0xffffu : 0xffff0000u, m[i][g] &= o ? 0xffffu : 0xffff0000u;
                                }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int g = 0; g < NG; g++) {
                            wide |= trx_a4p_wide(d[i][g], m[i][g]);
                            d[i][g] = trx_a4_hmul2(d[i][g], hv), m[i][g] = trx_a4_hmul2(m[i][g], hv);
                        }
                    if (wide) *(volatile int *)&s_wide = 1;
                    if (j >= 2) go = __all_sync(0xffffffffu, wait(&bar.v_empty[st], (j >> 1) - 1));
                    if (!go) break;
                    uint8_t *to = sv + st * S::K;
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        uint32_t x[4][4]; // [dim][position pair]
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            uint32_t h[4];
                            trx_a4_codes<true>(w[i][g], h);
#pragma unroll
                            for (int k = 0; k < 4; k++) x[k][i] = trx_a4_hfma2(h[k], d[i][g], m[i][g]);
                        }
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            *reinterpret_cast<uint4 *>(to + trx_a4p_chunk(32 * g + 4 * vn + k, t8, HD)) =
                                make_uint4(x[k][0], x[k][1], x[k][2], x[k][3]);
                    }
                    trx_fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) trx_a4p_arrive(&bar.v_full[st]);
                }
            }
        } else if (lane == 0) {
            // ---- products: O t += P t V of the tile before, then S t = Q t K
            const uint32_t aq = trx_smem(sq), ak = trx_smem(sk), av = trx_smem(sv);
            constexpr uint32_t is = S::IDESC | ((uint32_t)(KT >> 3) << 17), iv = S::IDESC | ((uint32_t)(HD >> 3) << 17);
            bool go = true;
            for (int j = 0; j <= n_all && go; j++) {
                for (int t = 0; t < 2 && go; t++) {
                    if (j > 0 && j - 1 < n_tiles[t]) {
                        const int st = (j - 1) & 1;
                        go = wait(&bar.p_ready[t], j - 1) && wait(&bar.v_full[st], (j - 1) >> 1);
                        if (!go) break;
                        trx_tc_fence_after();
#pragma unroll
                        for (int k = 0; k < KT / 16; k++)
                            trx_a4p_mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k,
                                           trx_umma_desc_sw128(av + st * S::K + (k >> 2) * (HD * 128) + 32 * (k & 3)), iv,
                                           j > 1 || k > 0);
                        if (j == n_tiles[t]) trx_umma_commit(&bar.o_full[t]);
                    }
                    if (j < n_tiles[t]) {
                        const int st = j & 1;
                        go = wait(&bar.k_full[st], j >> 1);
                        if (!go) break;
                        trx_tc_fence_after();
#pragma unroll
                        for (int k = 0; k < HD / 16; k++)
                            trx_a4p_mma(tmem + 128 * t, trx_umma_desc_sw128(aq + t * S::Q + (k >> 2) * (128 * 128) + 32 * (k & 3)),
                                        trx_umma_desc_sw128(ak + st * S::K + (k >> 2) * (KT * 128) + 32 * (k & 3)), is, k > 0);
                        trx_umma_commit(&bar.s_full[t]);
                    }
                }
                if (!go) break;
                if (j > 0) trx_umma_commit(&bar.v_empty[(j - 1) & 1]);
                if (j < n_all) trx_umma_commit(&bar.k_empty[j & 1]);
            }
            trx_umma_commit(&bar.done); // no product is in flight when the tensor memory goes
            wait(&bar.done, 0);
        }
        __syncwarp();
        trx_tc_fence_before();
        __syncthreads();
        trx_tc_fence_after();
        if (attempt > 0 || *(volatile int *)&s_wide == 0 || *(volatile int *)&s_fail != 0) break;
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
            for (int i = 0; i < 32; i += 4)
                trx_a4_out4<false>(io, out_at + 32 * g + i, make_float4(o[i] * x, o[i + 1] * x, o[i + 2] * x, o[i + 3] * x));
        }
        if (tid == 0 && s_fail) atomicCAS(a.err, 0, TRX_A4_GAVE_UP);
    }
    trx_tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        trx_tc_fence_after();
        trx_tmem_dealloc(s_tmem, 512);
    }
}
