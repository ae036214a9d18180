// fp8_matmul.cu — matrix product of e4m3 activations (a scale for each 128 of
// a row) with e4m3 weights (a scale for each block of 128 x 128).
//
//   y(c, r) = sum_b sx(c, b) * sw(r / 128, b) * sum_{k in block b} qx(c, k) * qw(r, k)
//
// The scale of a block is applied to its finished sum, so the inner sums are
// products of e4m3 values alone.
#include "../../include/cmolcu.h"
#include "fp8_weight.cuh"
#include "gemv_launch.cuh"

#include "tcgen05.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

struct Fp8MmArgs {
    Fp8W           w;
    const uint8_t *q;
    long long      q_ld;
    const float   *s;
    long long      s_ld, s_inc;
    int            n;
    void          *y;
    long long      y_ld;
};

// ---------------------------------------------------------------------------
// Up to 16 rows of activations: straight from memory
// ---------------------------------------------------------------------------
// Bound by the weights' stream, so what counts is that it divides evenly over the
// SMs and that nothing stands between a load and its use: no ring, no tensor
// memory, no cluster.  A warp takes 16 weight rows and every KW-th block of 128
// along k; what it loads (16 bytes a lane and row) is, as it lies in registers,
// the operand of the warp-wide product m16n8k32: the order of k within a block is
// the same permutation for both operands.  A block's product starts from zero and
// is scaled and added in f32.  The KW warps of the same rows add up through shared
// memory, in order.  6.2 us at 1x2048x11008 with weights from memory (3.6 TB/s; 4.5 us
// with the weight in L2), 2.1 at 1x960x2560.  k_fp8_mm_n with 16 columns takes 7.4 and 4.1
// there, but 10.1 us at 1x22016x2048 against 10.8: warps of more rows than a wave holds start
// their loads from nothing in every round.  Beyond 8 rows (two column groups) 100 to 204
// bytes a thread spill at 128 registers.
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int few_warps(int kw) { return kw > 8 ? kw : 8; }

template <int NG, int KW, typename TY>
__global__ void __launch_bounds__(32 * few_warps(KW), KW > 8 ? 1 : 2) k_fp8_mm_few(const Fp8MmArgs a) {
    constexpr int D = 2, W = few_warps(KW), RG = W / KW;                  // blocks in flight; warps, row groups of a CTA
    const Fp8W &w = a.w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kw = warp % KW, rg = warp / KW;
    const int g = lane >> 2, t = lane & 3;                                // row (column for b) and quarter of a fragment
    const int r0 = (blockIdx.x * RG + rg) * 16;                           // rows [r0, r0 + 16)
    const int nb = r0 < w.rows ? w.kblocks : 0;
    const uint8_t *wt = w.tiles + (size_t)(r0 >> 7) * nb * FP8_TILE_BYTES + ((r0 & 127) + g) * 128;
    const float *sw = w.scales + (size_t)(r0 >> 7) * nb;
    const int o0 = (t ^ g) << 4, o1 = ((t + 4) ^ g) << 4;                 // 16-byte chunks t and t + 4 of rows g, g + 8
    uint4 wr[D][4], x[D][NG][2];
    float s[D][NG][2], ws[D];
    auto load_w = [&](int d, int b) {
        if (b >= nb) return;
        const uint8_t *p = wt + (size_t)b * FP8_TILE_BYTES;
        wr[d][0] = ld_stream_u4(p + o0);
        wr[d][1] = ld_stream_u4(p + 1024 + o0);
        wr[d][2] = ld_stream_u4(p + o1);
        wr[d][3] = ld_stream_u4(p + 1024 + o1);
        ws[d] = sw[b];
    };
    auto load_x = [&](int d, int b) {
        if (b >= nb) return;
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const int c = 8 * j + g;
            const uint8_t *xp = a.q + c * a.q_ld + (long long)b * FP8_BLOCK + 16 * t;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                x[d][j][h] = make_uint4(0, 0, 0, 0);
                if (c < a.n && b * FP8_BLOCK + 64 * h + 16 * t < w.k) x[d][j][h] = *reinterpret_cast<const uint4 *>(xp + 64 * h);
                const int cc = 8 * j + 2 * t + h;                         // the column of accumulators h and 2 + h
                s[d][j][h] = a.s[min(cc, a.n - 1) * a.s_ld + b * a.s_inc];   // past the last column: not written
            }
        }
    };
    float acc[NG][4];
#pragma unroll
    for (int j = 0; j < NG; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
    for (int d = 0; d < D; d++) load_w(d, kw + d * KW);                   // weights do not wait for the previous kernel
    pdl_wait();
    pdl_launch_dependents();
#pragma unroll
    for (int d = 0; d < D; d++) load_x(d, kw + d * KW);
    for (int b0 = kw; b0 < nb; b0 += D * KW) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            if (b0 + d * KW >= nb) break;
#pragma unroll
            for (int j = 0; j < NG; j++) {
                float v[2][4] = {};
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint4 &p = wr[d][2 * h], &q = wr[d][2 * h + 1], &b = x[d][j][h];
                    mma_e4m3(v[h], p.x, q.x, p.y, q.y, b.x, b.y);
                    mma_e4m3(v[h], p.z, q.z, p.w, q.w, b.z, b.w);
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
                    acc[j][i] = __fmaf_rn(v[0][i] + v[1][i], s[d][j][i & 1] * ws[d], acc[j][i]);
            }
            load_w(d, b0 + (D + d) * KW);
            load_x(d, b0 + (D + d) * KW);
        }
    }
    __shared__ float part[W][8 * NG][16];
#pragma unroll
    for (int j = 0; j < NG; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) part[warp][8 * j + 2 * t + (i & 1)][g + 8 * (i >> 1)] = acc[j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < RG * 128 * NG; i += 32 * W) {    // (row group, column, row)
        const int r = i & 15, c = (i >> 4) % (8 * NG), gg = i / (128 * NG), row = (blockIdx.x * RG + gg) * 16 + r;
        float y = 0.f;
#pragma unroll
        for (int k = 0; k < KW; k++) y += part[gg * KW + k][c][r];
        if (row < w.rows && c < a.n) static_cast<TY *>(a.y)[c * a.y_ld + row] = fp8_t<TY>(y);
    }
}

// ---------------------------------------------------------------------------
// Few rows of activations: the weights' rows are the tensor core's M
// ---------------------------------------------------------------------------
// A CTA takes one row block of the weight (128 rows: the M of the product), NT
// activation rows (its N) and a range of k blocks.  Every block of 128 along k
// is a product of its own in tensor memory (four steps of K = 32); eight warps
// take it from there, multiply by the block's scales and add to sums in
// registers, while the tensor core forms the next blocks in other columns of
// tensor memory.
//
// Bound by the weights' stream (one byte a value, read once per NT activation
// rows): 16 KB blocks, contiguous along k, come by bulk copies into a ring.
// Where the row blocks are fewer than the SMs, k is split over the CTAs of a
// cluster.  Each owns some of the columns: the others store their sums into its
// ring, once its last product has read it (stores to another CTA are not waited
// for; loading them took longer than the rest of the sum), and after a barrier it
// adds them in the order of the split.
//
// Barriers, two a block as in k_fp8_mm_t: `full` counts both operands' bytes and
// the summing warps' release of tensor memory, `done` is the product's commit.
// Scales come eight blocks at a time.
//
// With weights from memory 9.3 us at 37x2048x11008 (eleven blocks a CTA; 8.6 with the weight
// in L2), 9.7 at 1x22016x2048 (NT = 16, 4.6 TB/s), 16.2 at 64x22016x2048 (NT = 64).
//
// Warps: 0 loads, 1 and 2 products in turn (1 also tensor memory), 3 scales, 4-11
// sums.
#define MMN_THREADS 384
#define MMN_SUM_WARPS 8
#define MMN_GROUP 8            // blocks whose scales come together
#define MMN_MAX_SPLIT 8        // CTAs of a cluster

struct Fp8MmnArgs {
    CUtensorMap tm_q;          // activations: [n][k] bytes, box 128 x NT, 128-byte swizzle
    Fp8MmArgs   a;
    int         ksplit;        // CTAs of a cluster
    int         kb_per;        // k blocks of a CTA
    int         own;           // columns of a CTA of a cluster (the last may have fewer)
    unsigned   *fault;
};

template <int NT>
struct MmnCfg {
    // Registers a thread where 32 columns' sums need more than two CTAs an SM leave (0: no split), of the first
    // warpgroup and of the summing warps.
    static constexpr int regs = NT == 64 ? 80 : 0, regs_few = 40, regs_sums = 96;
    static_assert(128 * regs_few + 256 * regs_sums <= 384 * 80, "register split");
    static constexpr int stage = FP8_TILE_BYTES + NT * FP8_BLOCK;
    static constexpr int scales = 2 * MMN_GROUP * NT * 4;
    static constexpr int stages = (110 * 1024 - 1024 - scales) / stage / 2 * 2;   // two CTAs an SM
    static constexpr int bufs = 4, cols = bufs * NT;                      // products in tensor memory
    static constexpr int smem = 1024 + stages * stage + scales;
    static_assert((NT + MMN_MAX_SPLIT) * FP8_BLOCK * 4 <= stages * stage, "ksplit * own columns fit in the ring");
    static_assert(stages >= bufs, "a buffer's release counts on a later block's stage");
};

template <int NT, typename TY>
__global__ void __launch_bounds__(MMN_THREADS, 2) k_fp8_mm_n(const __grid_constant__ Fp8MmnArgs p) {
    using Cfg = MmnCfg<NT>;
    constexpr int S = Cfg::stages, B = Cfg::bufs, C = NT / 2;             // C: columns of a summing warp
    constexpr int CH = C < 16 ? C : 16, NC = C / CH, G = MMN_GROUP;
    const Fp8W &w = p.a.w;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const long long c0 = (long long)blockIdx.x * NT;                      // first activation row
    const int ks = blockIdx.y, rb = blockIdx.z;
    const int b0 = ks * p.kb_per, nb = min(w.kblocks - b0, p.kb_per);     // k blocks [b0, b0 + nb), nb >= 1
    const int cols = (int)min((long long)NT, p.a.n - c0);

    uint8_t *base = reinterpret_cast<uint8_t *>(((uintptr_t)cmolcu_smem + 1023) & ~(uintptr_t)1023);
    float *scales = reinterpret_cast<float *>(base + S * Cfg::stage);     // [2 * G blocks][NT]
    float *part = reinterpret_cast<float *>(base);                        // [ksplit][own][128], over the drained ring
    __shared__ uint64_t full[S], done[S], sfull[2], sempty[2], drain;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;                                               // a bounded wait ran out: every role gives up
    volatile int *aborted = &s_abort;

    if (tid == 0) {
        t5_prefetch_map(&p.tm_q);
        for (int i = 0; i < S; i++) {
            mbar_init(&full[i], 1 + MMN_SUM_WARPS);
            mbar_init(&done[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sfull[i], 1);
            mbar_init(&sempty[i], MMN_SUM_WARPS);
        }
        mbar_init(&drain, 2);
        fence_mbar_init();
        s_abort = 0;
    }
    if (warp == 1) t5_alloc(&s_tmem, Cfg::cols);
    t5_fence_before();
    __syncthreads();
    t5_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();

    // A wait of a whole role: false when it, or another role's, ran out.
    auto wait = [&](uint64_t *bar, int parity, unsigned code) {
        if (mbar_try_wait(bar, parity)) return true;
        if (!*aborted && mbar_wait(bar, parity, p.fault, code)) return true;
        *aborted = 1;
        return false;
    };

    TY *y = static_cast<TY *>(p.a.y);
    const int r0 = rb * FP8_BLOCK;
    if (warp < 4) {
        if (Cfg::regs) t5_regs_dec<Cfg::regs_few>();
        if (warp == 0) {
            // ---- loads: the first weights do not wait for the previous kernel ----
            if (lane == 0) {
                const uint8_t *src = w.tiles + ((size_t)rb * w.kblocks + b0) * FP8_TILE_BYTES;
                auto load_w = [&](int st, int i) {
                    mbar_arrive_expect_tx(&full[st], Cfg::stage);
                    bulk_g2s(base + st * Cfg::stage, src + (size_t)i * FP8_TILE_BYTES, FP8_TILE_BYTES, &full[st]);
                };
                auto load_q = [&](int st, int i) {
                    t5_tma_2d(base + st * Cfg::stage + FP8_TILE_BYTES, &p.tm_q, (b0 + i) * FP8_BLOCK, (int)c0, &full[st]);
                };
                const int pre = min(S, nb);
                for (int i = 0; i < pre; i++) load_w(i, i);
                pdl_wait();                                                   // (and no bounded wait spans it)
                for (int i = 0; i < pre; i++) load_q(i, i);
                int st = 0, par = 0, i = pre;
                for (; i < nb; i++) {
                    if (!wait(&done[st], par, FAULT_GEMV_EMPTY)) break;
                    load_w(st, i);
                    load_q(st, i);
                    st++;
                    par ^= st == S;
                    st = st == S ? 0 : st;
                }
                if (*aborted)                                                 // what was issued lands before the CTA ends
                    for (int j = max(0, i - S); j < i; j++) mbar_wait(&full[j % S], (j / S) & 1, nullptr, 0);
            }
        } else if (warp == 1 || warp == 2) {
            // ---- products: warp 1 the even blocks, warp 2 the odd ones ----
            pdl_wait();
            if (lane == 0) {
                const uint32_t idesc = t5_idesc_e4m3(FP8_BLOCK, NT), lo = t5_desc_lo(smem_u32(base));
                int st = warp - 1, par = 0, buf = warp - 1;
                bool ready = false;                                           // this block's barrier was seen complete
                for (int i = warp - 1; i < nb; i += 2) {
                    if (!ready && !wait(&full[st], par, FAULT_GEMV_FULL)) break;
                    t5_fence_after();
                    const uint32_t da = lo + st * (Cfg::stage >> 4), db = da + (FP8_TILE_BYTES >> 4), d = tmem + buf * NT;
                    uint64_t *const f = &done[st];
                    st += 2;
                    par ^= st >= S;
                    st = st >= S ? st - S : st;
                    buf = (buf + 2) & (B - 1);
                    ready = mbar_test(&full[st], par);
                    t5_mma_e4m3<false>(d, da, db, idesc);
                    t5_mma_e4m3<true>(d, da + 2, db + 2, idesc);
                    t5_mma_e4m3<true>(d, da + 4, db + 4, idesc);
                    t5_mma_e4m3<true>(d, da + 6, db + 6, idesc);
                    t5_commit(f);
                }
                t5_commit(&drain);
            }
        } else if (warp == 3) {
            // ---- scales: activation scale x weight scale, a group's loads in flight together ----
            constexpr int L = (NT + 31) / 32;
            pdl_wait();
            const float *sw = w.scales + (size_t)rb * w.kblocks + b0;
            for (int i0 = 0, gi = 0; i0 < nb; i0 += G, gi++) {
                float v[G][L];
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int l = 0; l < L; l++) {
                        const int c = l * 32 + lane;
                        v[g][l] = i0 + g < nb && c < cols
                                      ? p.a.s[(c0 + c) * p.a.s_ld + (long long)(b0 + i0 + g) * p.a.s_inc] * sw[i0 + g]
                                      : 0.f;
                    }
                if (gi >= 2 && !__all_sync(0xffffffffu, wait(&sempty[gi & 1], ((gi >> 1) - 1) & 1, FAULT_GEMV_EMPTY))) break;
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int l = 0; l < L; l++)
                        if (l * 32 + lane < NT) scales[((gi & 1) * G + g) * NT + l * 32 + lane] = v[g][l];
                __syncwarp();
                if (lane == 0) mbar_arrive(&sfull[gi & 1]);
            }
        }
        __syncwarp();
        if (p.ksplit > 1) t5_cluster_sync();                                  // (the summing warps' arrival is what counts)
    } else {
        if (Cfg::regs) t5_regs_inc<Cfg::regs_sums>();
        // ---- sums: warp w has tensor-memory lanes 32 * (w % 4) .., half of the columns ----
        const int half = (warp - 4) >> 2;
        const uint32_t tcol = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + half * C;
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < B; i++) mbar_arrive(&full[i]);            // tensor memory is free
        pdl_wait();
        int st = 0, par = 0, buf = 0;
        bool ok = true;
        bool arrived = false;                                             // at the cluster's first barrier
        uint64_t acc[C / 2];                                              // sums of this lane's row, two columns each
#pragma unroll
        for (int i = 0; i < C / 2; i++) acc[i] = 0;
        uint32_t d[2][CH];
        // Block i, whose first CH columns are on their way to d[F]; before its last are added, the first of block
        // i + 1 are sent for.
        auto block = [&](auto first, int i) {
            constexpr int F = decltype(first)::value;
            if (i == nb - 1 && p.ksplit > 1) {                             // every product has read its operands
                __syncwarp();
                t5_cluster_arrive_all();
                arrived = true;
            }
            if (i % G == 0 && !__all_sync(0xffffffffu, wait(&sfull[(i / G) & 1], (i / (2 * G)) & 1, FAULT_GEMV_FULL))) {
                ok = false;
                return;
            }
            const float *sc = scales + (i % (2 * G)) * NT + half * C;
            uint64_t *const rel = &full[st + B >= S ? st + B - S : st + B];
            const uint32_t src = tcol + buf * NT;
            st++;
            par ^= st == S;
            st = st == S ? 0 : st;
            buf = (buf + 1) & (B - 1);
            bool ready = __all_sync(0xffffffffu, mbar_test(&done[st], par));
#pragma unroll
            for (int c = 0; c < NC; c++) {
                uint32_t(&dc)[CH] = d[(F + c) & 1], (&dn)[CH] = d[(F + c + 1) & 1];
                t5_wait_ld(dc);
                if (c < NC - 1) {
                    t5_ld(src + CH * (c + 1), dn);
                } else {
                    t5_fence_before();
                    t5_arrive(rel, lane == 0);
                    if (i + 1 < nb) {
                        if (!ready) ok = __all_sync(0xffffffffu, wait(&done[st], par, FAULT_GEMV_FULL));
                        t5_fence_after();
                        t5_ld(tcol + buf * NT, dn);
                    }
                }
#pragma unroll
                for (int j = 0; j < CH; j += 4) {
                    const ulonglong2 s4 = *reinterpret_cast<const ulonglong2 *>(sc + CH * c + j);
                    const int o = (CH * c + j) / 2;
                    acc[o] = t5_fma2(t5_pair(dc[j], dc[j + 1]), s4.x, acc[o]);
                    acc[o + 1] = t5_fma2(t5_pair(dc[j + 2], dc[j + 3]), s4.y, acc[o + 1]);
                }
            }
            if (i % G == G - 1) {
                __syncwarp();
                t5_arrive(&sempty[(i / G) & 1], lane == 0);
            }
        };
        ok = __all_sync(0xffffffffu, wait(&done[0], 0, FAULT_GEMV_FULL));
        t5_fence_after();
        t5_ld(tcol, d[0]);
        for (int i = 0; i < nb && ok; i += 2) {
            block(std::integral_constant<int, 0>(), i);
            if (ok && i + 1 < nb) block(std::integral_constant<int, (NC & 1)>(), i + 1);
        }
        __syncwarp();
        if (p.ksplit > 1) {
            if (!arrived) t5_cluster_arrive_all();
            t5_cluster_wait_all();
        }
        const int r = 32 * (warp & 3) + lane;
        if (p.ksplit == 1) {
            TY *yr = y + (c0 + half * C) * p.a.y_ld + r0 + r;
#pragma unroll
            for (int i = 0; i < C / 2; i++) {
                float v0, v1;
                t5_unpair(acc[i], v0, v1);
                if (r0 + r < w.rows) {
                    if (half * C + 2 * i < cols) yr[(long long)(2 * i) * p.a.y_ld] = fp8_t<TY>(v0);
                    if (half * C + 2 * i + 1 < cols) yr[(long long)(2 * i + 1) * p.a.y_ld] = fp8_t<TY>(v1);
                }
            }
        } else {
            // column c is the (c % own)-th of CTA c / own
            const uint32_t mine = smem_u32(part + (size_t)(ks * p.own) * FP8_BLOCK + r);
            int o = half * C / p.own, e = half * C % p.own;
#pragma unroll
            for (int i = 0; i < C / 2; i++) {
                float v[2];
                t5_unpair(acc[i], v[0], v[1]);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (half * C + 2 * i + h < cols) t5_cluster_st(t5_cluster_addr(mine + e * (FP8_BLOCK * 4), o), v[h]);
                    if (++e == p.own) { e = 0; o++; }
                }
            }
        }
    }
    __syncthreads();
    if (p.ksplit > 1) {
        t5_cluster_sync();
        // task = (column of this CTA, 4 rows)
        const int n_own = min(p.own, cols - ks * p.own);
        for (int t = tid; t < n_own * 32; t += MMN_THREADS) {
            const int col = t >> 5, rq = (t & 31) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int s = 0; s < p.ksplit; s++) {
                const float4 u = *reinterpret_cast<const float4 *>(part + (size_t)(s * p.own + col) * FP8_BLOCK + rq);
                v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
            }
            TY *yc = y + (c0 + ks * p.own + col) * p.a.y_ld + r0 + rq;
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (r0 + rq + j < w.rows) yc[j] = fp8_t<TY>(e[j]);
        }
    }
    if (tid == 0) mbar_wait(&drain, 0, p.fault, FAULT_GEMV_FULL);
    __syncthreads();
    if (warp == 1) {
        t5_fence_after();
        t5_dealloc(tmem, Cfg::cols);
    }
}

// ---------------------------------------------------------------------------
// Many rows of activations: they are the tensor core's M
// ---------------------------------------------------------------------------
// Two CTAs (a cluster on neighbouring SMs) form one tile of 256 activation rows
// x N weight rows: each holds half of both in shared memory, and every product
// of the pair (M = 256) reads both halves, so at N = 256 an SM loads 32 KB a block
// of 128 along k for work that takes its tensor core 512 clocks.  A lane of
// tensor memory is an activation row here, so a block's scale is one number a
// thread for every 128 columns: taking a block's product from tensor memory and
// adding it (128 columns a thread, two values an instruction) measured ~300
// clocks an SM alone, which hides behind the products.  (With the roles of the
// operands as in k_fp8_mm_n the scale differs from column to column and comes
// from shared memory: 670 clocks.)
//
// The CTAs are persistent: loads and products run on into the next tile while
// the sums of the last are written.  N is chosen so that the tiles fill the
// pairs of SMs evenly (mmt_launch).
//
// A wait or an arrival costs a thread about as much as two products cost it to
// issue, so two warps issue in turn, and there are two barriers a block: `full`
// counts the bytes of both CTAs' stages and the 16 summing warps' release of the
// part of tensor memory that the block will use, `done` (the products' commit,
// in both CTAs) frees the stage and hands the sums their block.
//
// 354 to 394 us at 8192x22016x2048 (N = 256) from one GPU to another (1.9 to 2.1 PFLOP/s, the
// tensor pipe half used; N = 128 takes 401 to 423): the summing warps take ~900 clocks a block of 256 columns,
// most of it waits for tensor memory one load after another.
//
// Warps: 0 loads, 1 and 3 products (rank 0), 2 tensor memory, 4-11 sums.
#define MMT_SUM_WARPS 8
#define MMT_THREADS (128 + 32 * MMT_SUM_WARPS)
// Registers a thread at launch, of the first warpgroup and of the summing warps.
#define MMT_REGS 168
#define MMT_REGS_FEW 40
#define MMT_REGS_SUMS 232
static_assert(128 * MMT_REGS_FEW + 32 * MMT_SUM_WARPS * MMT_REGS_SUMS == MMT_THREADS * MMT_REGS, "register split");

template <int N>
struct MmtCfg {
    static constexpr int rows = N / 2;                                      // weight rows of a CTA, columns of a sum
    static constexpr int group = 256 / N;                                   // blocks along k between two barriers
    static constexpr int block = FP8_TILE_BYTES + rows * FP8_BLOCK;
    static constexpr int stage = group * block;
    static constexpr int staging = MMT_SUM_WARPS * 2 * 32 * 64;             // a summing warp's way out: twice 32 rows x 64 bytes
    static constexpr int stages = (226 * 1024 - 1024 - staging) / stage / 2 * 2;
    static constexpr int smem = 1024 + stages * stage + staging;
    static_assert(N == 128 || N == 256, "a CTA's rows lie in one row block");
};

struct Fp8MmtArgs {
    CUtensorMap tm_q, tm_w;    // activations as above; weight tiles as rows of 128 bytes
    CUtensorMap tm_y;          // where vy: y, in boxes of 64 bytes x 32 rows, 64-byte swizzle
    Fp8MmArgs   a;
    int         mt, rt;        // tiles of activation rows and of weight rows
    int         vy;            // rows of y start on 16-byte boundaries: copies write y
    unsigned   *fault;
};

// Place of 16-byte chunk c of row lr in a half (32 rows x 64 bytes) of a summing
// warp's way out: the 64-byte swizzle of the TMA store, free of bank conflicts.
__device__ __forceinline__ int mmt_place(int lr, int c) { return lr * 64 + ((c ^ ((lr >> 1) & 3)) << 4); }

template <int N, typename TY>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MMT_THREADS, 1) k_fp8_mm_t(const __grid_constant__ Fp8MmtArgs p) {
    using Cfg = MmtCfg<N>;
    constexpr int S = Cfg::stages, B = 2, G = Cfg::group, R = Cfg::rows, CH = 32, NC = 128 / CH;
    static_assert(S % 2 == 0, "a stage belongs to one of the two issuing warps");
    const Fp8W &w = p.a.w;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)t5_cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const long long tiles = (long long)p.mt * p.rt;
    const int nb = w.kblocks, nr = (nb + G - 1) / G;    // blocks and groups of blocks along k

    uint8_t *base = reinterpret_cast<uint8_t *>(((uintptr_t)cmolcu_smem + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[S], done[S], drain;        // full: rank 0's counts
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    volatile int *aborted = &s_abort;

    if (tid == 0) {
        t5_prefetch_map(&p.tm_q);
        t5_prefetch_map(&p.tm_w);
        for (int i = 0; i < S; i++) {
            mbar_init(&full[i], 1 + 2 * MMT_SUM_WARPS);
            mbar_init(&done[i], 1);
        }
        mbar_init(&drain, 2);
        fence_mbar_init();
        s_abort = 0;
    }
    if (warp == 2) t5_alloc2(&s_tmem, 512);
    t5_fence_before();
    __syncthreads();
    t5_cluster_sync();                          // the other CTA's barriers are there
    t5_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();

    auto wait = [&](uint64_t *bar, int parity, unsigned code) {
        if (mbar_try_wait(bar, parity)) return true;
        if (!*aborted && mbar_wait(bar, parity, p.fault, code)) return true;
        *aborted = 1;
        return false;
    };

    if (warp < 4) {
        t5_regs_dec<MMT_REGS_FEW>();
        if (warp == 0 && lane == 0) {
            // ---- loads: this CTA's halves, counted on rank 0's barriers ----
            pdl_wait();
            int st = 0, use = 0;
            bool ok = true;
            for (long long t = pair; t < tiles && ok; t += pairs) {
                const int m = (int)(t % p.mt), r = (int)(t / p.mt);
                const int row = m * 256 + rank * 128, wrow = r * N + rank * R;
                for (int i = 0; i < nr; i++) {
                    if (use > 0 && !wait(&done[st], (use - 1) & 1, FAULT_GEMV_EMPTY)) {
                        ok = false;
                        break;
                    }
                    uint8_t *dst = base + st * Cfg::stage;
                    if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * Cfg::stage);
                    const uint32_t bar = t5_cluster_addr(smem_u32(&full[st]), 0);
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        // a block past the last: both operands lie past their tensors and read as zero
                        const int b = i * G + g, rb = b < nb ? wrow >> 7 : w.rblocks;
                        t5_tma2_2d(dst + g * Cfg::block, &p.tm_q, b * FP8_BLOCK, row, bar);
                        t5_tma2_2d(dst + g * Cfg::block + FP8_TILE_BYTES, &p.tm_w, 0,
                                   (rb * nb + (b < nb ? b : 0)) * FP8_BLOCK + (wrow & 127), bar);
                    }
                    if (++st == S) { st = 0; use++; }
                }
            }
            if (!ok && rank == 0)               // what was issued lands before the cluster ends
                for (int j = 0; j < S; j++) {
                    const int u = j < st ? use : use - 1;
                    if (u >= 0) mbar_wait(&full[j], u & 1, nullptr, 0);
                }
        } else if ((warp & 1) && lane == 0 && rank == 0) {
            // ---- products: warp 1 the even groups, warp 3 the odd ones ----
            pdl_wait();                         // so that no bounded wait spans the previous kernel
            const uint32_t idesc = t5_idesc_e4m3(256, N);
            const uint32_t lo = t5_desc_lo(smem_u32(base));
            const long long groups = (tiles - pair + pairs - 1) / pairs * nr;
            const uint32_t d = tmem + (warp >> 1) * 256;
            int st = warp >> 1, par = 0;
            bool ready = false;                 // this group's barrier was seen complete in the last round
            for (long long j = warp >> 1; j < groups; j += 2) {
                if (!ready && !wait(&full[st], par, FAULT_GEMV_FULL)) break;
                t5_fence_after();
                const uint32_t a0 = lo + st * (Cfg::stage >> 4);
                uint64_t *const f = &done[st];
                st += 2;
                par ^= st >= S;
                st = st >= S ? st - S : st;
                ready = mbar_test(&full[st], par);
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const uint32_t da = a0 + g * (Cfg::block >> 4), db = da + (FP8_TILE_BYTES >> 4);
                    t5_mma2_e4m3<false>(d + g * N, da, db, idesc);
                    t5_mma2_e4m3<true>(d + g * N, da + 2, db + 2, idesc);
                    t5_mma2_e4m3<true>(d + g * N, da + 4, db + 4, idesc);
                    t5_mma2_e4m3<true>(d + g * N, da + 6, db + 6, idesc);
                }
                t5_commit2(f);
            }
            t5_commit2(&drain);
        }
    } else {
        // ---- sums: lanes 32 * (warp % 4) .. are activation rows, R columns of a warp weight rows ----
        t5_regs_inc<MMT_REGS_SUMS>();
        const int half = (warp - 4) >> 2, lrow = rank * 128 + 32 * (warp & 3);
        const uint32_t tcol = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + half * R;
        const uint32_t full0 = t5_cluster_addr(smem_u32(&full[0]), 0);   // rank 0's, 8 bytes each
        uint8_t *const out = base + S * Cfg::stage + (warp - 4) * (2 * 32 * 64);
        int flip = 0;                                                     // which half of it
#pragma unroll
        for (int i = 0; i < B; i++) t5_cluster_arrive(full0 + 8 * i, lane == 0);   // tensor memory is free
        pdl_wait();
        int st = 0, par = 0, buf = 0;
        bool ok = true;
        // A tile's first rows, its scales' places and the scales of its first two groups, which are loaded before the
        // last tile is written.  Lanes past the last row and warps past the last block sum what they find and write
        // nothing.
        struct Tile {
            long long    row0;                                            // the warp's first activation row
            int          wrow;                                            // its first weight row
            const float *sx, *sw;
            float        x[2][G], w[2][G];
        };
        auto tile = [&](long long t) {
            Tile c;
            const int m = (int)(t % p.mt), r = (int)(t / p.mt);
            c.row0 = (long long)m * 256 + lrow;
            c.wrow = r * N + half * R;
            c.sx = p.a.s + min(c.row0 + lane, (long long)p.a.n - 1) * p.a.s_ld;
            c.sw = w.scales + (size_t)min(c.wrow >> 7, w.rblocks - 1) * nb;
#pragma unroll
            for (int j = 0; j < 2 * G; j++) {
                const int b = min(j, nb - 1);
                c.x[j / G][j % G] = c.sx[b * p.a.s_inc];
                c.w[j / G][j % G] = c.sw[b];
            }
            return c;
        };
        Tile nx = tile(pair);
        for (long long t = pair; t < tiles && ok; t += pairs) {
            const long long row0 = nx.row0;
            const int wrow = nx.wrow;
            const float *sx = nx.sx, *sw = nx.sw;
            float x[2][G], ws[2][G];
#pragma unroll
            for (int j = 0; j < 2 * G; j++) {
                x[j / G][j % G] = nx.x[j / G][j % G];
                ws[j / G][j % G] = nx.w[j / G][j % G];
            }
            uint64_t acc[R / 2];
#pragma unroll
            for (int j = 0; j < R / 2; j++) acc[j] = 0;
            uint32_t d[2][CH];
            // Group i of blocks, whose first 32 columns are on their way to d[0]; before its last 32 are added, the
            // first of group i + 1 are sent for.  xg and wg, its scales, were loaded two groups ago and their place
            // takes those of group i + 2.
            auto group = [&](int i, float (&xg)[G], float (&wg)[G]) {
                uint64_t s2[G];
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const float s = i * G + g < nb ? xg[g] * wg[g] : 0.f;
                    s2[g] = t5_pair(__float_as_uint(s), __float_as_uint(s));
                    const int b = min((i + 2) * G + g, nb - 1);
                    xg[g] = sx[b * p.a.s_inc];
                    wg[g] = sw[b];
                }
                // released for the group B groups on, which waits for this on its stage's barrier
                const uint32_t rel = full0 + 8 * (st + B >= S ? st + B - S : st + B), src = tcol + buf * 256;
                st++;
                par ^= st == S;
                st = st == S ? 0 : st;
                buf ^= 1;
                bool ready = false;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    uint32_t(&dc)[CH] = d[c & 1], (&dn)[CH] = d[(c + 1) & 1];
                    t5_wait_ld(dc);
                    if (c < NC - 1) {
                        t5_ld(src + (c + 1) * CH / R * N + (c + 1) * CH % R, dn);
                        if (c == NC - 2) ready = __all_sync(0xffffffffu, mbar_test(&done[st], par));
                    } else {
                        t5_fence_before();
                        t5_cluster_arrive(rel, lane == 0);
                        if (i + 1 < nr) {
                            if (!ready) ok = __all_sync(0xffffffffu, wait(&done[st], par, FAULT_GEMV_FULL));
                            t5_fence_after();
                            t5_ld(tcol + buf * 256, dn);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < CH / 2; j++)
                        acc[c * CH % R / 2 + j] =
                            t5_fma2(t5_pair(dc[2 * j], dc[2 * j + 1]), s2[c * CH / R], acc[c * CH % R / 2 + j]);
                }
            };
            ok = __all_sync(0xffffffffu, wait(&done[st], par, FAULT_GEMV_FULL));
            t5_fence_after();
            t5_ld(tcol + buf * 256, d[0]);
            for (int i = 0; i < nr && ok; i += 2) {
                group(i, x[0], ws[0]);
                if (ok && i + 1 < nr) group(i + 1, x[1], ws[1]);
            }
            if (t + pairs < tiles) nx = tile(t + pairs);
            if (!ok || wrow >= w.rows) continue;
            // ---- out: 64 bytes of each of the warp's 32 rows at a time, through shared memory ----
            // A copy out ends at y's last column only in whole 16 bytes (it wrote into what lies between the rows), so the
            // last box goes value by value where the columns' bytes are not a multiple of that.
            constexpr int E = 64 / (int)sizeof(TY), V = 16 / (int)sizeof(TY);   // columns a pass, a 16-byte chunk
            const int by_copy = !p.vy ? 0 : w.rows % V ? w.rows / E * E : w.rows;   // columns that copies write
#pragma unroll
            for (int ps = 0; ps < R / E; ps++) {
                uint8_t *const stg = out + flip * (32 * 64);
                flip ^= 1;
                const int col0 = wrow + ps * E;
                if (p.vy) {                                               // the copy out of this half, two passes ago
                    if (lane == 0) t5_tma_store_wait_read<1>();
                    __syncwarp();
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    alignas(16) TY v[V];
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        float lo, hi;
                        t5_unpair(acc[(ps * E + c * V + e) / 2], lo, hi);
                        v[e] = fp8_t<TY>(lo);
                        v[e + 1] = fp8_t<TY>(hi);
                    }
                    *reinterpret_cast<uint4 *>(stg + mmt_place(lane, c)) = *reinterpret_cast<uint4 *>(v);
                }
                if (p.vy) {
                    t5_fence_proxy();
                    __syncwarp();
                    if (lane == 0) {
                        if (col0 < by_copy && row0 < p.a.n) t5_tma_store_2d(&p.tm_y, col0, (int)row0, stg);
                        t5_tma_store_commit();                            // one group a pass, as the wait counts them
                    }
                }
                __syncwarp();
                // the other columns: 32 consecutive values of a row an instruction (f32: two passes'), eight rows in
                // flight
                constexpr int PP = 32 / E;
                if (by_copy < w.rows && ps % PP == PP - 1 && col0 + E > by_copy) {
                    const int c0 = col0 - (PP - 1) * E + lane, e = lane % E;
                    const uint8_t *const src = PP == 1 ? stg : out + (lane / E) * (32 * 64);
                    const int rows = c0 >= by_copy && c0 < w.rows ? (int)min((long long)32, p.a.n - row0) : 0;
                    TY *y = static_cast<TY *>(p.a.y) + row0 * p.a.y_ld + c0;
                    for (int b = 0; b < 32; b += 8) {
                        TY v[8];
#pragma unroll
                        for (int u = 0; u < 8; u++)
                            v[u] = reinterpret_cast<const TY *>(src + mmt_place(b + u, e / V))[e % V];
#pragma unroll
                        for (int u = 0; u < 8; u++) {
                            if (b + u < rows) *y = v[u];
                            y += p.a.y_ld;
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (p.vy && lane == 0) t5_tma_store_wait_all();
    }
    __syncwarp();
    t5_fence_before();
    __syncthreads();
    if (tid == 0) mbar_wait(&drain, 0, p.fault, FAULT_GEMV_FULL);        // the last arrival from rank 0's products
    __syncwarp();
    t5_cluster_sync();                          // neither CTA's memory is in use by the other any more
    if (warp == 2) {
        t5_fence_after();
        t5_dealloc2(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// cuTensorMapEncodeTiled, reached through the runtime's driver entry point (no
// link-time dependency on the driver library).
typedef CUresult (*encode_t)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                             const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static encode_t encode_fn() {
    static const encode_t fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<encode_t>(f);
    }();
    return fn;
}

// Activations as [n][k] bytes, read in boxes of `rows` rows x 128 bytes with
// the 128-byte swizzle; what lies past n or k reads as zero.
static bool q_map(CUtensorMap *m, const Fp8MmArgs &a, int rows) {
    const encode_t enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)a.w.k, (cuuint64_t)a.n};
    const cuuint64_t strides[1] = {(cuuint64_t)a.q_ld};
    const cuuint32_t box[2] = {FP8_BLOCK, (cuuint32_t)rows}, es[2] = {1u, 1u};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(a.q), dims, strides, box, es,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Sets kernel k's shared memory once on each device, and checks that it was built
// with `regs` registers a thread (0: any number).
template <typename K>
static cudaError_t kernel_ready(std::atomic<int> (&ready)[64], K k, size_t smem, int regs) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (ready[dev]) return cudaSuccess;
    cudaFuncAttributes fa = {};
    e = cudaFuncGetAttributes(&fa, k);
    if (e == cudaSuccess && regs && fa.numRegs != regs) e = cudaErrorInvalidConfiguration;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) ready[dev] = 1;
    return e;
}

// Launch with programmatic dependent launch and a (1, cluster, 1) cluster.
template <typename P>
static cudaError_t mm_launch(void (*k)(P), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st,
                             const P &p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 1;
    at[1].val.clusterDim.y = cluster;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, p);
}

// Warps that share a row group's k: 32 warps an SM (us at 1, 2, 4, 8, 16 warps a row group: 22016x2048 12.0, 12.5, 10.9,
// 11.0, 15.8; 2048x11008 33.6, 16.7, 9.2, 5.3, 4.8; 49152x2048 21.6, 19.7, 19.5, 21.2, 33.1).
static int few_split(const Fp8MmArgs &a) {
    const int groups = (a.w.rows + 15) / 16;
    int kw = 1;
    while (kw < 16 && (long long)groups * kw < device_sm_count() * 32LL && kw * 2 <= a.w.kblocks) kw *= 2;
    return kw;
}

template <int NG, typename TY>
static cudaError_t few_launch(const Fp8MmArgs &a, cudaStream_t st) {
    const int groups = (a.w.rows + 15) / 16, kw = few_split(a), wc = few_warps(kw);
    const dim3 grid((groups * kw + wc - 1) / wc), block(32 * wc);
    switch (kw) {
    case 1: return launch_k(k_fp8_mm_few<NG, 1, TY>, grid, block, 0, st, true, a);
    case 2: return launch_k(k_fp8_mm_few<NG, 2, TY>, grid, block, 0, st, true, a);
    case 4: return launch_k(k_fp8_mm_few<NG, 4, TY>, grid, block, 0, st, true, a);
    case 8: return launch_k(k_fp8_mm_few<NG, 8, TY>, grid, block, 0, st, true, a);
    default: return launch_k(k_fp8_mm_few<NG, 16, TY>, grid, block, 0, st, true, a);
    }
}

// CTAs that share k and their blocks each: a power of two that does not more than fill
// most of one wave at two an SM (96x2048x11008 at 6 CTAs 17.5 us, at 4 14.4; 16x2048x11008
// at 16 15.6, at 8 7.3), less those that the rounding up of their blocks leaves without
// any (12 blocks over 8: 6 CTAs of 2).  Giving all of the power of two CTAs one block
// fewer or more measured no better (16 / 32 / 64 columns, us: 37x576x1536 3.8, 4.1, 4.7 against 3.6, 4.1,
// 4.8; 64x960x2560 5.8, 4.9, 5.8 against 5.3, 5.0, 6.3; 24x2048x1152 5.2, 4.2, 5.0 against 4.1, 4.0,
// 5.1).
static int mmn_split(const Fp8MmArgs &a, int nt, int &kb_per) {
    const long long ctas = ((a.n - 1) / nt + 1) * (long long)a.w.rblocks, slots = device_sm_count() * 7LL / 4;
    int ks = 1;
    while (ks < MMN_MAX_SPLIT && ks * 2 <= a.w.kblocks && ctas * ks * 2 <= slots) ks *= 2;
    kb_per = (a.w.kblocks + ks - 1) / ks;
    return (a.w.kblocks + kb_per - 1) / kb_per;
}

template <int NT, typename TY>
static cudaError_t mmn_launch(const Fp8MmArgs &a, unsigned *fault, cudaStream_t st) {
    using Cfg = MmnCfg<NT>;
    Fp8MmnArgs p = {};
    p.a = a;
    p.fault = fault;
    static std::atomic<int> ready[64];
    const cudaError_t e = kernel_ready(ready, k_fp8_mm_n<NT, TY>, Cfg::smem, Cfg::regs);
    if (e != cudaSuccess) return e;
    if (!q_map(&p.tm_q, a, NT)) return cudaErrorInvalidValue;
    const long long tiles = (a.n - 1) / NT + 1;
    p.ksplit = mmn_split(a, NT, p.kb_per);
    p.own = (int)((std::min<long long>(a.n, NT) + p.ksplit - 1) / p.ksplit);
    const dim3 grid((unsigned)tiles, p.ksplit, a.w.rblocks);
    return mm_launch(k_fp8_mm_n<NT, TY>, grid, MMN_THREADS, Cfg::smem, p.ksplit, st, p);
}

// Weight tiles as rows of 128 bytes, read `rows` at a time (their bytes are in
// the operand's swizzled order already); row blocks past the last read as zero.
static bool w_map(CUtensorMap *m, const Fp8W &w, int rows) {
    const encode_t enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {FP8_BLOCK, (cuuint64_t)w.rblocks * w.kblocks * FP8_BLOCK};
    const cuuint64_t strides[1] = {FP8_BLOCK};
    const cuuint32_t box[2] = {FP8_BLOCK, (cuuint32_t)rows}, es[2] = {1u, 1u};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(w.tiles), dims, strides, box, es,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// y, written in boxes of 64 bytes x 32 rows; rows past it are left alone, and columns in
// whole 16 bytes.
template <typename TY>
static bool y_map(CUtensorMap *m, const Fp8MmArgs &a) {
    const encode_t enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)a.w.rows, (cuuint64_t)a.n};
    const cuuint64_t strides[1] = {(cuuint64_t)a.y_ld * sizeof(TY)};
    const cuuint32_t box[2] = {64 / (cuuint32_t)sizeof(TY), 32}, es[2] = {1u, 1u};
    const CUtensorMapDataType t = std::is_same<TY, float>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : std::is_same<TY, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return enc(m, t, 2, a.y, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int N, typename TY>
static cudaError_t mmt_launch(const Fp8MmArgs &a, unsigned *fault, cudaStream_t st) {
    using Cfg = MmtCfg<N>;
    const auto kern = k_fp8_mm_t<N, TY>;
    Fp8MmtArgs p = {};
    p.a = a;
    p.fault = fault;
    if (!q_map(&p.tm_q, a, FP8_BLOCK) || !w_map(&p.tm_w, a.w, Cfg::rows)) return cudaErrorInvalidValue;
    p.mt = (a.n - 1) / 256 + 1;
    p.rt = (a.w.rows - 1) / N + 1;
    p.vy = fp8_vec(a.y, a.y_ld * (long long)sizeof(TY)) > 0;
    if (p.vy && !y_map<TY>(&p.tm_y, a)) return cudaErrorInvalidValue;
    // the register split of the kernel adds up only to what it was built with
    static std::atomic<int> ready[64];
    const cudaError_t e = kernel_ready(ready, kern, Cfg::smem, MMT_REGS);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)p.mt * p.rt;
    const int pairs = (int)std::min<long long>(tiles, device_sm_count() / 2);
    return launch_k(kern, dim3(2 * pairs), dim3(MMT_THREADS), Cfg::smem, st, true, p);
}

// Which form, by what it is estimated to take (us, fitted to 18 weights of 0.9 to 67 MB at 1
// to 8192 rows, each call with another weight so that they come from memory):
//   k_fp8_mm_few            1.4 + 0.5 a round of CTAs + the larger of 0.20 a MB of weights (0.34 beyond 8 rows, where
//                           registers are spilled) and 1.0 (2.0) a block along k of a warp beyond the two in flight
//   k_fp8_mm_n, 16 / 32 / 64   2.3 / 2.4 / 3.0, at two CTAs an SM 0.55 / 0.75 / 1.5 and with a split of k 1.05 / 1.15 /
//                           1.3 more; 0.26 / 0.32 / 0.59 a block of 128 along k and 2.2 / 2.6 / 3.4 between rounds of
//                           CTAs (f32 0.1 / 0.2 / 0.4 more); 0.077 / 0.076 / 0.04 a MB of weights
//   k_fp8_mm_t, 128 / 256   3.6 / 3.8; a round of tiles 0.245 / 0.485 a block of 128 along k where it is the only
//                           one, else 0.27 / 0.49, and 0.85 / 1.6 more; where rows of y do not start on 16-byte
//                           boundaries 1.1 / 2.8 on top (f32 3.1 / 5.9), which hides from 4 blocks along k on
// Of 376 measured calls, 9 take a form that is more than 6 % slower than the best (26 % at 64x2049x8192); all lose 0.5 %
// together, and 475 calls of other sizes 1.0 %.  Measured, for instance (few; 16, 32, 64; 128, 256):
//   1x960x2560  2.1; 4.1, 4.3, 5.3; -        1x22016x2048  10.9; 10.1, 11.9, 14.5; -
//   16x5760x960  4.5; 4.7, 5.0, 6.3; -       16x11008x2048  9.5; 7.5, 8.4, 11; -
//   64x2048x2048  -; 5.5, 5.9, 7.3; 7.9, 12  128x2048x11008  -; 17, 12.6, 14.4; 24.6, 44
//   256x22016x2048  -; 70, 43, 39; 18.6, 22  512x22016x2048  -; 134, 83, 65; 29.1, 30.8
//   1024x22016x2048  -; 55, 51               8192x22016x2048  -; 401, 367
//   4096x16383x128 bf16, y unaligned  -; -; 65, 72 (aligned 42, 31)
static int mm_form(const Fp8MmArgs &a, bool aligned, int elem_bytes) {
    static const struct { int nt; double fixed, two, split, block, round, mb; } mmn[3] = {
        {16, 2.3, 0.55, 1.05, 0.26, 2.2, 0.077}, {32, 2.4, 0.75, 1.15, 0.32, 2.6, 0.076}, {64, 3.0, 1.5, 1.3, 0.59, 3.4, 0.04}};
    static const struct { int n; double fixed, one, more, tile, out16, out32; } mmt[2] = {
        {128, 3.6, 0.245, 0.27, 0.85, 1.1, 3.1}, {256, 3.8, 0.485, 0.49, 1.6, 2.8, 5.9}};
    const int sms = device_sm_count(), kb = a.w.kblocks;
    const double mb = 1e-6 * a.w.rows * a.w.k;
    double best = 1e30;
    int form = 0;
    auto take = [&](int f, double t) {
        if (t < best) { best = t; form = f; }
    };
    if (a.n <= 16) {
        const int kw = few_split(a), wc = few_warps(kw), slots = kw > 8 ? sms : 2 * sms;
        const int ctas = ((a.w.rows + 15) / 16 * kw + wc - 1) / wc;
        const int chain = (kb + kw - 1) / kw - 2;
        take(CMOLCU_FP8_FEW, 1.4 + 0.5 * ((ctas - 1) / slots + 1) +
                                 (a.n <= 8 ? std::max(0.20 * mb, 1.0 * chain) : std::max(0.34 * mb, 2.0 * chain)));
    }
    for (const auto &f : mmn) {
        int kb_per;
        const long long ks = mmn_split(a, f.nt, kb_per), ctas = ((a.n - 1) / f.nt + 1) * (long long)a.w.rblocks * ks;
        const double rounds = (double)((ctas - 1) / (2 * sms) + 1);
        const double round = f.round + (elem_bytes == 4 ? 0.006 * f.nt : 0);
        take(f.nt, f.fixed + (ctas > sms ? f.two : 0) + (ks > 1 ? f.split : 0) + rounds * kb_per * f.block +
                       (rounds - 1) * round + f.mb * mb);
    }
    const long long mt = (a.n - 1) / 256 + 1, pairs = std::max(1, sms / 2);
    for (const auto &f : mmt) {
        const long long rounds = (mt * ((a.w.rows - 1) / f.n + 1) - 1) / pairs + 1;
        const double out = aligned ? 0 : (elem_bytes == 2 ? f.out16 : f.out32) * std::min(1.0, 4.0 / kb);
        take(f.n, f.fixed + rounds * (kb * (rounds == 1 ? f.one : f.more) + f.tile + out));
    }
    return form;
}

template <typename TY>
static cudaError_t mm_run(int form, const Fp8MmArgs &a, unsigned *fault, cudaStream_t st) {
    switch (form) {
    case CMOLCU_FP8_FEW: return a.n <= 8 ? few_launch<1, TY>(a, st) : few_launch<2, TY>(a, st);
    case 16: return mmn_launch<16, TY>(a, fault, st);
    case 32: return mmn_launch<32, TY>(a, fault, st);
    case 64: return mmn_launch<64, TY>(a, fault, st);
    case 128: return mmt_launch<128, TY>(a, fault, st);
    default: return mmt_launch<256, TY>(a, fault, st);
    }
}

static int matmul(const char *who, int form, const cmolcu_fp8_weight_t *w, const void *q, long long q_ld,
                  const float *scales, long long s_ld, long long s_inc, int n, void *y, int y_dtype, long long y_ld,
                  void *stream) {
    if (!w) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    if (n < 0 || n > 1 << 30) { cmolcu_set_error("%s: n=%d", who, n); return -1; }
    if (!fp8_elem_bytes(y_dtype)) { cmolcu_set_error("%s: unsupported dtype %d", who, y_dtype); return -1; }
    if (n == 0) return 0;
    if (!q || !scales || !y) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    if (fp8_misaligned(who, scales, 4) || fp8_misaligned(who, y, fp8_elem_bytes(y_dtype))) return -1;
    if (n == 1) {                                       // a single row has no stride
        q_ld = (w->w.k + 15) / 16 * 16;
        y_ld = (w->w.rows + 15LL) / 16 * 16;
    }
    if ((reinterpret_cast<uintptr_t>(q) & 15) || q_ld < w->w.k || q_ld % 16) {
        cmolcu_set_error("%s: q rows must start on 16-byte boundaries (q_ld=%lld)", who, q_ld);
        return -1;
    }
    if (y_ld < w->w.rows) { cmolcu_set_error("%s: rows of y overlap (y_ld=%lld)", who, y_ld); return -1; }
    Fp8Device dev(w->device);
    FP8_TRY(who, dev.err);
    Fp8MmArgs a = {};
    a.w = w->w;
    a.q = static_cast<const uint8_t *>(q); a.q_ld = q_ld;
    a.s = scales; a.s_ld = s_ld; a.s_inc = s_inc;
    a.n = n; a.y = y; a.y_ld = y_ld;
    const int yb = fp8_elem_bytes(y_dtype);
    if (!form) form = mm_form(a, fp8_vec(y, y_ld * yb) > 0, yb);
    unsigned *fault = cmolcu_fault_word(w->device);
    const cudaStream_t st = (cudaStream_t)stream;
    FP8_TRY(who, fp8_with_type(y_dtype, [&](auto t) {
        return mm_run<decltype(t)>(form, a, fault, st);
    }));
    return 0;
}

extern "C" int cmolcu_fp8_matmul(const cmolcu_fp8_weight_t *w, const void *q, long long q_ld, const float *scales,
                                 long long s_ld, long long s_inc, int n, void *y, int y_dtype, long long y_ld,
                                 void *stream) {
    return matmul("cmolcu_fp8_matmul", 0, w, q, q_ld, scales, s_ld, s_inc, n, y, y_dtype, y_ld, stream);
}

extern "C" int cmolcu_fp8_matmul_form(const cmolcu_fp8_weight_t *w, int n) {
    if (!w || n < 1 || n > 1 << 30) return 0;
    Fp8Device dev(w->device);
    Fp8MmArgs a = {};
    a.w = w->w;
    a.n = n;
    return mm_form(a, true, 4);
}

extern "C" int cmolcu_fp8_matmul_as(int form, const cmolcu_fp8_weight_t *w, const void *q, long long q_ld,
                                    const float *scales, long long s_ld, long long s_inc, int n, void *y, int y_dtype,
                                    long long y_ld, void *stream) {
    static const char *who = "cmolcu_fp8_matmul_as";
    if (form != CMOLCU_FP8_FEW && form != 16 && form != 32 && form != 64 && form != 128 && form != 256) {
        cmolcu_set_error("%s: no form %d", who, form);
        return -1;
    }
    if (form == CMOLCU_FP8_FEW && n > 16) { cmolcu_set_error("%s: n=%d is too many for form %d", who, n, form); return -1; }
    return matmul(who, form, w, q, q_ld, scales, s_ld, s_inc, n, y, y_dtype, y_ld, stream);
}
