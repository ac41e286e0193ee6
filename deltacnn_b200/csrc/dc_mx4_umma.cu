// Product of two MXFP4 matrices on the block-scaled tensor core path: out[t][f] = sum_k a[t][k] b[f][k] + bias[f], a with
// `m` rows (tokens), b with `n` rows (features, a weight in nn.Linear's layout), both packed along k (dc_mx4.cuh).
//
// tcgen05.mma kind::mxf4 multiplies 128 rows of one operand by up to 256 rows of the other, 64 values of k at a time, applies
// the two scale bytes of each row's blocks in the multiplier and adds in float32 in tensor memory. The FEATURES are the 128
// rows here and the tokens the columns of the accumulator: few tokens are then a narrow accumulator (16 columns for one
// token) instead of 128 rows of padding, a thread of the epilogue owns one feature (one bias value), and the 32 lanes of a
// warp store 32 neighbouring features of a token.
//
// A step is 256 values of k: one TMA box per operand (rows of 128 bytes, 128-byte swizzle) and the step's two 512-byte scale
// tiles per 128 rows, in one contiguous copy each; tcgen05.cp spreads a scale tile over the four lane quarters of tensor
// memory. Roles: one thread issues the copies, one the scale copies and MMAs, four warps drain accumulators; persistent CTAs,
// two accumulators.
//
// dc_mx4_linear on few tokens packs them in the same kernel: eight warps quantise a step's rows straight into the stage, in the
// swizzled layout that the TMA would have written, and arrive on the stage's barrier beside the copies.
//
// Bound: many tokens, the tensor core and the shared memory that feeds it; few tokens, the weight's bytes. Then the tiles
// do not fill the GPU, and the CTAs of a cluster share a tile along k: each leaves its float32 sums in its own shared
// memory, and after a cluster barrier every CTA adds a share of the columns in the order of the ranks (same bits every time).
// Measured (bf16, device time): 8192 x 4096 -> 14336 196 us = 4.9 PFLOP/s (four times the measured bf16 rate is 6.7; 217 us in a
// loop of seconds, at the power limit); 1 x 4096 -> 14336 10 us for 31 MB of weight (4.8 us at the copy rate; launch, tensor
// memory, first and last round trips are the rest).
#include <cstring>
#include "dc_umma.cuh"
#include "dc_mx4.cuh"

namespace dc {

__device__ int g_mx4_error = 0;

constexpr int kMxThreads = 192;            // TMA warp, MMA warp, four epilogue warps
constexpr int kMxQuantThreads = 320;       // with the tokens quantised on the way: eight warps for that, four of them drain
constexpr int kMxQuantRounds = 2;          // rounds of eight warps that dc_mx4_linear spends on packing inside the product, at most
constexpr int kMxStep = 256;               // values of k per step: one 128-byte row
constexpr uint32_t kMxTmem = 512;
// A cluster's CTAs wait for one another: they ask for an SM's whole shared memory, so that no CTA of another kernel that waits in a
// cluster too can hold tensor memory on the same SM while its peer waits for theirs.
constexpr int kWholeSmem = 226 * 1024;

// Columns (tokens) per tile -> stages of the ring, accumulators, tensor memory columns of a stage's scales.
template <int NT> struct MxCfg {
    static constexpr int kB = NT * 128;
    static constexpr int kStage = kABytes + kB + 2048;
    static constexpr int kStages = NT == 128 ? 6 : 8;
    static constexpr int kScCols = 16;
    static constexpr int kSmem = kStages * kStage + 1024;
    static_assert(2 * NT + kStages * kScCols <= (int)kMxTmem, "tensor memory");
    static_assert(kSmem <= 227 * 1024 - 1024, "shared memory");
};

struct MxGemmParams {
    const uint8_t *a_sc, *b_sc;            // scales of the tokens, of the features
    const void* x;                         // tokens in the result's type, where they are quantised on the way
    int k, access, groups;                 // their width; bytes a read of theirs may take; groups of eight rows
    const void* bias;
    void* out;
    int64_t m;
    int n, nb, tiles_k, steps;             // blocks, scale tiles and steps along k
    int tiles_f, tiles;                    // feature tiles, all tiles
    int bias_dtype, out_dtype;
    int out_even;                          // out is 4-byte aligned (16-bit results)
};

struct MxPlan {
    bool pair, quant;
    int nt, split;
    int64_t tiles;
};

__device__ __forceinline__ uint64_t mx_scale_desc(uint32_t smem_addr) {
    uint64_t d = 0;                                       // rows of 16 bytes, 8-row groups 128 bytes apart, no swizzle
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)(128 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    return d;
}
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// kind::mxf4: A and B e2m1 (format 1) K-major, scales ue8m0 (bit 23), M = 128 (1 in bits 27-28), N = n; the scale data id of
// either operand (bits 29-30, 4-5) picks the half of a 32-bit scale word: 0 or 2.
__host__ __device__ constexpr uint32_t mx_idesc(int n) { return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | (1u << 27); }
__host__ __device__ constexpr uint32_t mx_idesc2(int n) { return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | (2u << 27); }      // M = 256
__device__ __forceinline__ uint32_t mx_idesc_half(uint32_t half) { return (half << 30) | (half << 5); }      // half * 2 in bits 29-30 and 4-5

template <typename OT> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Hands an accumulator back. Relaxed: what has to be ordered before it are tensor memory reads (waited for and fenced by the
// caller); a release would also wait for the stores of the tile before (1100 cycles measured).
__device__ __forceinline__ void cluster_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float mx_bias(const MxGemmParams& p, int f) {
    if (p.bias == nullptr) return 0.f;
    if (p.bias_dtype == DC_F32) return ((const float*)p.bias)[f];
    if (p.bias_dtype == DC_F16) return __half2float(((const __half*)p.bias)[f]);
    return __bfloat162float(((const __nv_bfloat16*)p.bias)[f]);
}

template <typename OT, int NT, bool SPLIT, bool QUANT>
__global__ void __launch_bounds__(QUANT ? kMxQuantThreads : kMxThreads, 1) k_mx4_gemm(const MxGemmParams p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b) {
    using Cfg = MxCfg<NT>;
    constexpr int S = Cfg::kStages;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[2 * S + 4];
    __shared__ uint32_t s_u32[2];
    volatile uint32_t* ok_flag = &s_u32[1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (S + s); };
    auto acc_full = [&](int a) { return bar0 + 8u * (2 * S + a); };
    auto acc_empty = [&](int a) { return bar0 + 8u * (2 * S + 2 + a); };
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(full(s), QUANT ? 1 + p.groups : 1); mbar_init(empty(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(acc_full(a), 1); mbar_init(acc_empty(a), 4); }
        *ok_flag = 1;
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc(smem_u32(&s_u32[0]), kMxTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_u32[0];
    const uint32_t tmem_sc = tmem + 2 * NT;
    grid_dep_launch();
    grid_dep_wait();

    // this CTA's steps of every tile: all of them, or (SPLIT) its rank's share
    const int rank = SPLIT ? (int)blockIdx.y : 0, ranks = SPLIT ? (int)gridDim.y : 1;
    const int k_lo = (int)((int64_t)p.steps * rank / ranks), k_hi = (int)((int64_t)p.steps * (rank + 1) / ranks);

    if (warp == 0) {
        // ---- copies: tokens' and features' boxes and scales of a step into a stage
        int issued = 0;
        if (elect_one()) {
            int s = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
                const int tf = tile % p.tiles_f, tt = tile / p.tiles_f;
                for (int ks = k_lo; ks < k_hi; ++ks) {
                    if (!mbar_wait(empty(s), phase ^ 1u, ok_flag)) { *ok_flag = 0; atomicExch(&g_mx4_error, 1); ok = false; break; }
                    const uint32_t at = ring + s * Cfg::kStage;
                    const int nsc = min(2, p.tiles_k - ks * 2);
                    mbar_expect_tx(full(s), (uint32_t)(kABytes + nsc * 512 + (QUANT ? 0 : Cfg::kB + nsc * 512)));
                    tma_load_rows(at, &map_b, ks * 128, tf * 128, full(s));
                    bulk_g2s(at + kABytes + Cfg::kB, p.b_sc + ((int64_t)tf * p.tiles_k + ks * 2) * 512, (uint32_t)nsc * 512u, full(s));
                    if constexpr (!QUANT) {
                        tma_load_rows(at + kABytes, &map_a, ks * 128, tt * NT, full(s));
                        bulk_g2s(at + kABytes + Cfg::kB + 1024, p.a_sc + ((int64_t)tt * NT / 128 * p.tiles_k + ks * 2) * 512, (uint32_t)nsc * 512u, full(s));
                    }
                    ++issued;
                    if (++s == S) { s = 0; phase ^= 1u; }
                }
            }
            if (!ok) {       // leave no copy in flight behind
                const int last = issued < S ? issued : S;
                for (int i = issued - last; i < issued; ++i)
                    for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(full(i % S), (uint32_t)(i / S) & 1u); ++w) {}
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- scales to tensor memory, MMAs
        if (elect_one()) {
            int s = 0, it = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x, ++it) {
                const int a = it & 1, use = it >> 1;
                if (!mbar_wait(acc_empty(a), (uint32_t)(use & 1) ^ 1u, ok_flag)) { *ok_flag = 0; atomicExch(&g_mx4_error, 2); break; }
                tc_fence_after();
                const uint32_t d = tmem + a * NT;
                for (int ks = k_lo; ks < k_hi; ++ks) {
                    if (!mbar_wait(full(s), phase, ok_flag)) { *ok_flag = 0; atomicExch(&g_mx4_error, 3); ok = false; break; }
                    tc_fence_after();
                    const uint32_t at = ring + s * Cfg::kStage, sc = tmem_sc + s * Cfg::kScCols;
                    const int nsc = min(2, p.tiles_k - ks * 2);
                    for (int q = 0; q < nsc; ++q) {
                        tmem_cp_scales(sc + q * 4, mx_scale_desc(at + kABytes + Cfg::kB + q * 512));
                        tmem_cp_scales(sc + 8 + q * 4, mx_scale_desc(at + kABytes + Cfg::kB + 1024 + q * 512));
                    }
                    const uint64_t da = make_smem_desc(at), db = make_smem_desc(at + kABytes);
                    const int chunks = min(4, (p.nb - ks * 8 + 1) >> 1);          // 64 values of k each
                    for (int c = 0; c < chunks; ++c)
                        umma_mxf4(d, da + c * 2, db + c * 2, mx_idesc(NT) | mx_idesc_half(c & 1), sc + (c >> 1) * 4,
                                  sc + 8 + (c >> 1) * 4, (ks > k_lo || c > 0) ? 1u : 0u);
                    umma_commit(empty(s));
                    if (++s == S) { s = 0; phase ^= 1u; }
                }
                if (ok) umma_commit(acc_full(a));
            }
        }
        __syncwarp();
    } else {
        // ---- accumulators out: warp w owns lanes 32 (w % 4) .. + 31, a lane is a feature
        const int quarter = warp & 3;
        int it = 0;
        [[maybe_unused]] uint32_t seq = 0;         // steps so far
        // A wait that ran out: a tile that is shared along k becomes NaN in the columns of every rank, instead of a sum without
        // this rank's share. (The accumulator of a failed copy or MMA never arrives, so that the draining warps come through here.)
        [[maybe_unused]] auto spoil = [&] {
            float* part = reinterpret_cast<float*>(raw + (ring - smem_u32(raw)));
            for (int c = 0; c < NT; ++c) part[c * 128 + quarter * 32 + lane] = __uint_as_float(0x7fffffffu);
        };
        for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x, ++it) {
            const int a = it & 1, use = it >> 1;
            const int tf = tile % p.tiles_f, tt = tile / p.tiles_f;
            if constexpr (QUANT) {
                // A step's 256 values of every token, straight into the stage, in groups of eight rows; groups of a step and
                // steps go round the eight warps. A warp has the eight rows' reads in flight; a lane takes eight values of a
                // row, 16-byte pieces in the 128-byte swizzle, the scales of four blocks as one word of the scale tile.
                const int64_t row0 = (int64_t)tt * NT;
                const int rows = (int)(p.m - row0 < NT ? p.m - row0 : NT);
                bool ok = true;
                for (int ks = k_lo; ks < k_hi && ok; ++ks, ++seq) {
                    const int s = (int)(seq % S);
                    uint8_t* codes = raw + (ring - smem_u32(raw)) + s * Cfg::kStage + kABytes;
                    for (int g = 0; g < p.groups; ++g) {
                        if ((int)((seq * p.groups + g) & 7u) != warp - 2) continue;
                        const int64_t col = (int64_t)ks * kMxStep + lane * 8;
                        Eight<OT> v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int r = g * 8 + j;
                            const OT* row = (const OT*)p.x + (row0 + r) * p.k;
                            const int64_t end = r < rows ? p.k : 0;
                            if (p.access == 16) v[j].template load<16>(row, col, end);
                            else if (p.access == 4) v[j].template load<4>(row, col, end);
                            else v[j].template load<(int)sizeof(OT)>(row, col, end);
                        }
                        if (!mbar_wait_warp(empty(s), ((uint32_t)(seq / S) & 1u) ^ 1u, ok_flag)) { *ok_flag = 0; atomicExch(&g_mx4_error, 9); ok = false; break; }
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int r = g * 8 + j;
                            if (r >= rows) break;
                            uint32_t sb;
                            *reinterpret_cast<uint32_t*>(codes + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = mx4_encode_lane<OT>(v[j], sb);
                            const uint32_t word = mx4_scale_quad(sb, lane);
                            if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(codes + Cfg::kB + 1024 + (lane >> 4) * 512 + (r & 31) * 16 + (r >> 5) * 4) = word;
                        }
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(full(s));
                    }
                }
                if (!ok) {
                    if constexpr (SPLIT) if (warp < 6) spoil();
                    break;
                }
                if (warp >= 6) continue;
            }
            const int f = tf * 128 + quarter * 32 + lane;
            const float bias = f < p.n && !SPLIT ? mx_bias(p, f) : 0.f;
            if (!mbar_wait_warp(acc_full(a), (uint32_t)(use & 1), ok_flag)) {
                *ok_flag = 0;
                atomicExch(&g_mx4_error, 4);
                if constexpr (SPLIT) spoil();
                break;
            }
            tc_fence_after();
            const uint32_t src = tmem + a * NT + ((uint32_t)quarter << 21);
            const int64_t t0 = (int64_t)tt * NT;
            const int cols = (int)(p.m - t0 < NT ? p.m - t0 : NT);
            for (int c = 0; c < NT; c += 16) {
                uint32_t r[16];
                tmem_ld16(src + c, r);
                tmem_ld_wait();
                if constexpr (SPLIT) {
                    float* part = reinterpret_cast<float*>(raw + (ring - smem_u32(raw)));        // the stages are free: every MMA has read its own
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[(c + i) * 128 + quarter * 32 + lane] = __uint_as_float(r[i]);
                } else if (f < p.n) {
                    OT* o = (OT*)p.out + (t0 + c) * p.n + f;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (c + i < cols) o[(int64_t)i * p.n] = from_f<OT>(__uint_as_float(r[i]) + bias);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(a));
        }
    }
    if constexpr (SPLIT) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        // columns rank, rank + ranks, ... of the tile: sum over the ranks in their order
        const int tile = blockIdx.x, tf = tile % p.tiles_f, tt = tile / p.tiles_f;
        const int64_t t0 = (int64_t)tt * NT;
        const int cols = (int)(p.m - t0 < NT ? p.m - t0 : NT);
        // four features at a time, every rank's share of them in flight together
        const int mine = 32 * ((cols - rank + ranks - 1) / ranks);
        for (int i = threadIdx.x; i < mine; i += blockDim.x) {
            const int col = rank + (i >> 5) * ranks, f = tf * 128 + (i & 31) * 4;
            float4 x[8];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < ranks) {
                    uint32_t remote;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(ring + (uint32_t)(col * 128 + (i & 31) * 4) * 4u), "r"(q));
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[q].x), "=f"(x[q].y), "=f"(x[q].z), "=f"(x[q].w) : "r"(remote) : "memory");
                }
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < ranks) { v[0] += x[q].x; v[1] += x[q].y; v[2] += x[q].z; v[3] += x[q].w; }
            OT* o = (OT*)p.out + (t0 + col) * p.n + f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (f + j < p.n) o[j] = from_f<OT>(v[j] + mx_bias(p, f + j));
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, kMxTmem);
}

// ---------------------------------------------------------------------------------------------
// Many tokens: two SMs per tile
// ---------------------------------------------------------------------------------------------
// A cluster of two CTAs computes 256 features x 256 tokens with tcgen05.mma.cta_group::2: either CTA holds 128 features and
// stages its features' rows and HALF of the tokens' rows, the tensor cores read the other half from the peer. Per step an SM
// stages 32 KB of codes for 128 x 256 outputs instead of 48 KB. Either CTA's copies count on the leader's barrier, the
// leader issues the scale copies and MMAs for both, its commits arrive in both.
// The accumulator takes 256 of the 512 columns and the stages' scales 120, so there is one accumulator; the epilogue (eight
// warps, a thread holds 128 tokens of its feature) therefore first drains it into registers, hands it back, and
// stores while the next tile's MMAs run. Lanes hold neighbouring features of one token pair per register: a shuffle with the
// neighbour lane makes four-byte stores of two features where the row width is even.
// Measured: a step takes 0.36-0.39 us whatever it multiplies (128, 192 or 256 tokens: about 150 cycles an MMA, 18 a scale copy),
// so 256 tokens it is: with 128 or 192, which have room for two accumulators, 8192 x 4096 -> 14336 takes 314 and 234 us
// (196). Issuing the MMAs from a warp-uniform loop instead of one lane's changes nothing (202). What sets those 150 cycles is not
// known: the tensor pipe counts 56 % active, L2 38 % of its rate, DRAM 14 %, and leaving the operands' copies out gains 4 %.
constexpr int kM2Threads = 320;            // TMA warp, MMA warp, eight epilogue warps
constexpr int kM2Stages = 5;
constexpr int kM2Tok = 256;                // tokens of a tile (128 rows staged per CTA)
constexpr int kM2Stage = kABytes + kABytes + 1024 + 2048;
constexpr int kM2ScCols = 24;
constexpr int kM2Smem = kM2Stages * kM2Stage + 1024;
static_assert(kM2Smem <= kWholeSmem, "shared memory");
static_assert(kM2Stage % 1024 == 0, "stages are swizzle-aligned");
static_assert(kM2Tok + kM2Stages * kM2ScCols <= (int)kMxTmem, "tensor memory");

__device__ __forceinline__ void tma2_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void umma2_mxf4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem2_cp_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Arrives on the barrier at this offset in both CTAs once everything issued so far has been executed.
__device__ __forceinline__ void umma2_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename OT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kM2Threads, 1)
k_mx4_gemm2(const MxGemmParams p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
            const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb) {
    constexpr int S = kM2Stages;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[2 * S + 2];
    __shared__ uint32_t s_u32[2];
    volatile uint32_t* ok_flag = &s_u32[1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };              // used in the leader only
    auto empty = [&](int s) { return bar0 + 8u * (S + s); };
    const uint32_t acc_full = bar0 + 8u * (2 * S), acc_empty = bar0 + 8u * (2 * S + 1);      // the latter in the leader only
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 16);
        *ok_flag = 1;
        fence_barrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_u32[0])), "r"(kMxTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s_u32[0];
    const uint32_t tmem_sc = tmem + kM2Tok;
    grid_dep_launch();
    grid_dep_wait();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (warp == 0) {
        if (elect_one()) {
            int s = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = pair; tile < p.tiles && ok; tile += pairs) {
                const int tf = tile % p.tiles_f, tt = tile / p.tiles_f;
                for (int ks = 0; ks < p.steps; ++ks) {
                    if (!mbar_wait(empty(s), phase ^ 1u, ok_flag)) { *ok_flag = 0; atomicExch(&g_mx4_error, 5); ok = false; break; }
                    const uint32_t at = ring + s * kM2Stage;
                    // the leader's barrier, where the copies of both CTAs count: in a pair's shared window the leader's addresses are
                    // those with bit 24 clear
                    const uint32_t bar = full(s) & 0xFEFFFFFFu;
                    if (rank == 0) mbar_expect_tx(full(s), 2 * kM2Stage);
                    tma2_load(at, &map_b, ks * 128, tf * 256 + (int)rank * 128, bar);
                    tma2_load(at + kABytes, &map_a, ks * 128, tt * kM2Tok + (int)rank * 128, bar);
                    // two scale tiles of this CTA's features, two of either half of the tokens
                    tma2_load(at + 2 * kABytes, &map_sb, 0, (tf * 2 + (int)rank) * p.tiles_k + ks * 2, bar);
                    tma2_load(at + 2 * kABytes + 1024, &map_sa, 0, tt * 2 * p.tiles_k + ks * 2, bar);
                    tma2_load(at + 2 * kABytes + 2048, &map_sa, 0, (tt * 2 + 1) * p.tiles_k + ks * 2, bar);
                    ++issued;
                    if (++s == S) { s = 0; phase ^= 1u; }
                }
            }
            if (!ok && rank == 0) {       // leave no copy in flight behind, the peer's included
                const int last = issued < S ? issued : S;
                for (int i = issued - last; i < issued; ++i)
                    for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(full(i % S), (uint32_t)(i / S) & 1u); ++w) {}
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            int s = 0;
            uint32_t phase = 0, use = 0;
            bool ok = true;
            for (int tile = pair; tile < p.tiles && ok; tile += pairs, use ^= 1u) {
                if (!mbar_wait(acc_empty, use ^ 1u, ok_flag)) { *ok_flag = 0; atomicExch(&g_mx4_error, 6); break; }
                tc_fence_after();
                for (int ks = 0; ks < p.steps; ++ks) {
                    if (!mbar_wait(full(s), phase, ok_flag)) { *ok_flag = 0; atomicExch(&g_mx4_error, 7); ok = false; break; }
                    tc_fence_after();
                    const uint32_t at = ring + s * kM2Stage, sc = tmem_sc + s * kM2ScCols;
                    const int nsc = min(2, p.tiles_k - ks * 2);
                    for (int q = 0; q < nsc; ++q) {
                        tmem2_cp_scales(sc + q * 4, mx_scale_desc(at + 2 * kABytes + q * 512));
                        tmem2_cp_scales(sc + 8 + q * 8, mx_scale_desc(at + 2 * kABytes + 1024 + q * 512));
                        tmem2_cp_scales(sc + 8 + q * 8 + 4, mx_scale_desc(at + 2 * kABytes + 2048 + q * 512));
                    }
                    const uint64_t da = make_smem_desc(at), db = make_smem_desc(at + kABytes);
                    const int chunks = min(4, (p.nb - ks * 8 + 1) >> 1);
                    for (int c = 0; c < chunks; ++c)
                        umma2_mxf4(tmem, da + c * 2, db + c * 2, mx_idesc2(kM2Tok) | mx_idesc_half(c & 1), sc + (c >> 1) * 4, sc + 8 + (c >> 1) * 8,
                                   (ks > 0 || c > 0) ? 1u : 0u);
                    umma2_commit(empty(s));
                    if (++s == S) { s = 0; phase ^= 1u; }
                }
                if (ok) umma2_commit(acc_full);
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const uint32_t acc_empty_leader = cluster_addr(acc_empty, 0);
        uint32_t use = 0;
        for (int tile = pair; tile < p.tiles; tile += pairs, use ^= 1u) {
            const int tf = tile % p.tiles_f, tt = tile / p.tiles_f;
            const int f = tf * 256 + (int)rank * 128 + quarter * 32 + lane;
            const float bias = f < p.n ? mx_bias(p, f) : 0.f;
            if (!mbar_wait_warp(acc_full, use, ok_flag)) { *ok_flag = 0; atomicExch(&g_mx4_error, 8); break; }
            tc_fence_after();
            const uint32_t src = tmem + half * 128 + ((uint32_t)quarter << 21);
            const int64_t t0 = (int64_t)tt * kM2Tok + half * 128;
            const int cols = (int)(p.m - t0 < 128 ? p.m - t0 : 128);          // may be negative: nothing to store
            OT* o = (OT*)p.out + t0 * p.n + f;
            if constexpr (sizeof(OT) == 4) {
                uint32_t r[128];
#pragma unroll
                for (int c = 0; c < 128; c += 16) tmem_ld16(src + c, *reinterpret_cast<uint32_t(*)[16]>(&r[c]));
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) cluster_arrive(acc_empty_leader);
                if (f < p.n) {
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c < cols) o[(int64_t)c * p.n] = __uint_as_float(r[c]) + bias;
                }
            } else {
                uint32_t r[64];          // tokens 2 i (low half) and 2 i + 1 of this lane's feature
                {
                    uint32_t v[8][16];
#pragma unroll
                    for (int c = 0; c < 8; ++c) tmem_ld16(src + c * 16, v[c]);
                    tmem_ld_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) cluster_arrive(acc_empty_leader);
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        r[i] = pack2<OT>(__uint_as_float(v[i >> 3][(2 * i) & 15]) + bias, __uint_as_float(v[i >> 3][(2 * i + 1) & 15]) + bias);
                }
                if ((p.n & 1) == 0 && p.out_even) {
                    const int odd = lane & 1;
                    uint32_t* o2 = reinterpret_cast<uint32_t*>(o - odd + (int64_t)odd * p.n);
                    const int64_t step = p.n;          // two rows, in words
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        const uint32_t q = __shfl_xor_sync(DC_FULL, r[i], 1);
                        const uint32_t v = odd ? __byte_perm(q, r[i], 0x7632) : __byte_perm(r[i], q, 0x5410);
                        if (2 * i + odd < cols && f < p.n) o2[i * step] = v;          // f and its neighbour are in or out together
                    }
                } else if (f < p.n) {
                    uint16_t* o1 = reinterpret_cast<uint16_t*>(o);
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        if (2 * i < cols) o1[(int64_t)(2 * i) * p.n] = (uint16_t)r[i];
                        if (2 * i + 1 < cols) o1[(int64_t)(2 * i + 1) * p.n] = (uint16_t)(r[i] >> 16);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();          // no arrival, copy or MMA of the pair is outstanding behind this
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kMxTmem) : "memory");
}

// Packed matrix [rows][16 nb] bytes as a tensor map, box 128 bytes x `box_rows`, 128-byte swizzle.
typedef CUresult (*MxEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static MxEncodeFn mx_encoder() {
    static const MxEncodeFn fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            return reinterpret_cast<MxEncodeFn>(ptr);
        (void)cudaGetLastError();
        return (MxEncodeFn) nullptr;
    }();
    return fn;
}
// The encoder needs a context; a thread that has not called the runtime yet gets the current device's one and a second try.
template <typename F> static bool mx_encode(F&& encode) {
    if (encode() == CUDA_SUCCESS) return true;
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess && encode() == CUDA_SUCCESS;
}
static bool encode_mx4_map(CUtensorMap* map, const void* data, int64_t rows, int64_t row_bytes, int box_rows) {
    const MxEncodeFn fn = mx_encoder();
    if (fn == nullptr) return false;
    const cuuint64_t gdim[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
    const cuuint64_t gstride[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {128u, (cuuint32_t)box_rows};
    const cuuint32_t estride[2] = {1u, 1u};
    return mx_encode([&] {
        return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(data), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
}

// The scale tiles as rows of 128 words, a box of two consecutive tiles along k.
static bool encode_mx4_scales(CUtensorMap* map, const void* scales, int64_t tiles) {
    const MxEncodeFn fn = mx_encoder();
    if (fn == nullptr) return false;
    const cuuint64_t gdim[2] = {128u, (cuuint64_t)tiles};
    const cuuint64_t gstride[1] = {512u};
    const cuuint32_t box[2] = {128u, 2u};
    const cuuint32_t estride[2] = {1u, 1u};
    return mx_encode([&] {
        return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(scales), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
}

template <typename OT>
static int launch_mx4_pair(const MxGemmParams& p, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& msa, const CUtensorMap& msb, cudaStream_t st) {
    static PerDeviceOnce once;
    bool* set = once.slot();
    if (set == nullptr) return DC_ERR_LAUNCH;
    if (!*set) {
        if (cudaFuncSetAttribute(k_mx4_gemm2<OT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWholeSmem) != cudaSuccess) return check_launch();
        *set = true;
    }
    const int pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1;
    return launch_pdl(k_mx4_gemm2<OT>, dim3((unsigned)(2 * (p.tiles < pairs ? p.tiles : pairs))), dim3(kM2Threads), kWholeSmem, st, p, ma, mb, msa, msb);
}

template <typename OT, int NT, bool SPLIT, bool QUANT>
static int launch_mx4(const MxGemmParams& p, int split, const CUtensorMap& ma, const CUtensorMap& mb, cudaStream_t st) {
    constexpr size_t smem = SPLIT ? (size_t)kWholeSmem : (size_t)MxCfg<NT>::kSmem;
    static PerDeviceOnce once;
    bool* set = once.slot();
    if (set == nullptr) return DC_ERR_LAUNCH;
    if (!*set) {
        if (cudaFuncSetAttribute(k_mx4_gemm<OT, NT, SPLIT, QUANT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return check_launch();
        *set = true;
    }
    const int sms = sm_count();
    const dim3 grid((unsigned)(SPLIT ? p.tiles : p.tiles < sms ? p.tiles : sms), (unsigned)split);
    return launch_pdl_cluster(k_mx4_gemm<OT, NT, SPLIT, QUANT>, grid, dim3(QUANT ? kMxQuantThreads : kMxThreads), smem, st, split, p, ma, mb);
}

template <typename OT, bool SPLIT>
static int launch_mx4_nt(int nt, const MxGemmParams& p, int split, const CUtensorMap& ma, const CUtensorMap& mb, cudaStream_t st) {
    if (p.x != nullptr) {
        switch (nt) {
            case 16: return launch_mx4<OT, 16, SPLIT, true>(p, split, ma, mb, st);
            case 32: return launch_mx4<OT, 32, SPLIT, true>(p, split, ma, mb, st);
            default: return launch_mx4<OT, 64, SPLIT, true>(p, split, ma, mb, st);
        }
    }
    switch (nt) {
        case 16: return launch_mx4<OT, 16, SPLIT, false>(p, split, ma, mb, st);
        case 32: return launch_mx4<OT, 32, SPLIT, false>(p, split, ma, mb, st);
        case 64: return launch_mx4<OT, 64, SPLIT, false>(p, split, ma, mb, st);
        default: break;
    }
    if constexpr (SPLIT) return launch_mx4<OT, 128, SPLIT, false>(p, split, ma, mb, st);
    else return DC_ERR_UNSUPPORTED;          // 128 tokens a tile: clusters only
}
template <typename OT>
static int launch_mx4_split(const MxPlan& pl, const MxGemmParams& p, const CUtensorMap& ma, const CUtensorMap& mb, cudaStream_t st) {
    return pl.split > 1 ? launch_mx4_nt<OT, true>(pl.nt, p, pl.split, ma, mb, st) : launch_mx4_nt<OT, false>(pl.nt, p, 1, ma, mb, st);
}

// How a product is cut: pairs of SMs, or tiles of nt tokens, each by one CTA or shared along k by `split`; quant: dc_mx4_linear
// quantises the tokens inside the product.
static MxPlan mx4_plan(int64_t m, int64_t n, int64_t k) {
    const int sms = sm_count();
    const int steps = (int)divup64(k, kMxStep);
    MxPlan pl{};
    pl.split = 1;
    // columns of a tile: no more than the tokens need
    pl.nt = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
    pl.tiles = divup64(n, 128) * divup64(m, pl.nt);
    // tiles that leave most SMs idle are shared along k by a cluster of up to 8 CTAs, at least one step each (clusters of 8 take
    // the SMs of a GPC by halves: more than a dozen do not run at once, 200 x 2048 -> 1000 took 11.4 us with 16)
    while (pl.split < 8 && pl.tiles * pl.split * 2 <= sms && steps >= pl.split * 2 && (pl.split < 4 || pl.tiles <= 12)) pl.split *= 2;
    // More than 64 tokens: pairs of SMs (5.3 us and 0.39 us a step for one tile each), unless a cluster saves seven steps and more.
    // Pairs / clusters: 128 x 256 -> 256 5.6 / 8.4 us, 1024 x 1024 -> 1024 7.0 / 8.4, 128 x 4096 -> 14336 (no room for clusters) 12.2 /
    // 14.2, 200 x 4096 -> 4096 11.6 / 10.8, 128 x 4096 -> 4096 11.6 / 8.4, 4096 x 8192 -> 256 17.5 / 13.7.
    pl.pair = m > 64 && steps - steps / pl.split < 7;
    if (pl.pair) {
        pl.tiles = divup64(n, 256) * divup64(m, kM2Tok);
        return pl;
    }
    // Quantising inside makes every feature tile's CTA read the tokens unpacked: eight rows of a step and warp at a time, which
    // waits for their 1 us of latency in every round of the eight warps. Device time inside / with a launch of its own (2.2 us of
    // it), bf16: one round, 1 x 4096 -> 14336, 10.0 / 11.8 us; two, 8 x 4096 -> 14336, 11.4 / 11.7, and 64 x 1280 -> 1000, 12.3 /
    // 11.5 (but a call of the host costs 5 us less); four, 16 x 4096 -> 14336, 16.4 / 12.1.
    const int64_t rounds = divup64(divup64(pl.tiles, sms) * divup(steps, pl.split) * divup64(m, 8), 8);
    pl.quant = m <= 64 && rounds <= kMxQuantRounds;
    return pl;
}

// x != NULL: the tokens unpacked, in the result's type; a_data / a_scales otherwise.
static int mx4_product(const void* x, const void* a_data, const void* a_scales, const void* b_data, const void* b_scales, const void* bias, void* out, int64_t m,
                       int64_t n, int64_t k, int bias_dtype, int out_dtype, cudaStream_t st) {
    const MxPlan pl = mx4_plan(m, n, k);
    if (pl.tiles > 0x7fffff00LL || (divup64(m > n ? m : n, 128) + 2) * mx4_scale_tiles(k) > 0x7fffff00LL) return DC_ERR_SHAPE;
    MxGemmParams p{};
    p.a_sc = (const uint8_t*)a_scales; p.b_sc = (const uint8_t*)b_scales; p.bias = bias; p.out = out;
    p.m = m; p.n = (int)n; p.nb = (int)mx4_blocks(k); p.tiles_k = (int)mx4_scale_tiles(k); p.steps = (int)divup64(k, kMxStep);
    p.bias_dtype = bias_dtype; p.out_dtype = out_dtype;
    p.out_even = (reinterpret_cast<uintptr_t>(out) & 3u) == 0;
    p.tiles_f = (int)divup64(n, pl.pair ? 256 : 128);
    p.tiles = (int)pl.tiles;
    p.x = x; p.k = (int)k; p.groups = (int)divup64(m < 64 ? m : 64, 8);
    p.access = out_dtype == DC_F32 ? row_access<float>(x, k) : row_access<__half>(x, k);
    alignas(64) CUtensorMap ma, mb;
    if (!encode_mx4_map(&mb, b_data, n, (int64_t)p.nb * 16, 128)) return DC_ERR_UNSUPPORTED;
    if (x != nullptr) ma = mb;          // not read
    else if (!encode_mx4_map(&ma, a_data, m, (int64_t)p.nb * 16, pl.pair ? kM2Tok / 2 : pl.nt)) return DC_ERR_UNSUPPORTED;
    if (pl.pair) {
        alignas(64) CUtensorMap msa, msb;
        if (!encode_mx4_scales(&msa, a_scales, divup64(m, 128) * p.tiles_k) || !encode_mx4_scales(&msb, b_scales, divup64(n, 128) * p.tiles_k)) return DC_ERR_UNSUPPORTED;
        switch (out_dtype) {
            case DC_F32: return launch_mx4_pair<float>(p, ma, mb, msa, msb, st);
            case DC_F16: return launch_mx4_pair<__half>(p, ma, mb, msa, msb, st);
            default: return launch_mx4_pair<__nv_bfloat16>(p, ma, mb, msa, msb, st);
        }
    }
    switch (out_dtype) {
        case DC_F32: return launch_mx4_split<float>(pl, p, ma, mb, st);
        case DC_F16: return launch_mx4_split<__half>(pl, p, ma, mb, st);
        default: return launch_mx4_split<__nv_bfloat16>(pl, p, ma, mb, st);
    }
}

static bool mx4_sizes_ok(int64_t m, int64_t n, int64_t k) {
    return m >= 0 && n >= 0 && k > 0 && m <= 0x7ffff000LL && n <= 0x7ffff000LL && k <= 0x7ffff000LL;
}

int mx4_error_code() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_mx4_error, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace dc

using namespace dc;

extern "C" {

int dc_mx4_matmul(const void* a_data, const void* a_scales, const void* b_data, const void* b_scales, const void* bias, void* out, int64_t m, int64_t n,
                  int64_t k, int32_t bias_dtype, int32_t out_dtype, void* stream) {
    if (!mx4_sizes_ok(m, n, k)) return DC_ERR_SHAPE;
    if (out_dtype < DC_F32 || out_dtype > DC_BF16 || (bias != nullptr && (bias_dtype < DC_F32 || bias_dtype > DC_BF16))) return DC_ERR_DTYPE;
    if (m == 0 || n == 0) return DC_OK;
    if (a_data == nullptr || a_scales == nullptr || b_data == nullptr || b_scales == nullptr || out == nullptr) return DC_ERR_NULL_POINTER;
    if (!aligned16(a_data) || !aligned16(a_scales) || !aligned16(b_data) || !aligned16(b_scales)) return DC_ERR_ALIGNMENT;
    return mx4_product(nullptr, a_data, a_scales, b_data, b_scales, bias, out, m, n, k, bias_dtype, out_dtype, (cudaStream_t)stream);
}

size_t dc_mx4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (!mx4_sizes_ok(m, n, k) || m == 0 || n == 0 || mx4_plan(m, n, k).quant) return 0;
    return dc_mx4_data_bytes(m, k) + dc_mx4_scale_bytes(m, k);
}

int dc_mx4_linear(const void* x, const void* w_data, const void* w_scales, const void* bias, void* out, int64_t m, int64_t n, int64_t k, int32_t dtype,
                  int32_t bias_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (!mx4_sizes_ok(m, n, k)) return DC_ERR_SHAPE;
    if (dtype < DC_F32 || dtype > DC_BF16 || (bias != nullptr && (bias_dtype < DC_F32 || bias_dtype > DC_BF16))) return DC_ERR_DTYPE;
    if (m == 0 || n == 0) return DC_OK;
    if (x == nullptr || w_data == nullptr || w_scales == nullptr || out == nullptr) return DC_ERR_NULL_POINTER;
    if (!aligned16(w_data) || !aligned16(w_scales) || !aligned16(workspace)) return DC_ERR_ALIGNMENT;
    if (mx4_plan(m, n, k).quant)
        return mx4_product(x, nullptr, nullptr, w_data, w_scales, bias, out, m, n, k, bias_dtype, dtype, (cudaStream_t)stream);
    if (workspace == nullptr) return DC_ERR_NULL_POINTER;
    const size_t data = dc_mx4_data_bytes(m, k);
    if (workspace_bytes < data + dc_mx4_scale_bytes(m, k)) return DC_ERR_WORKSPACE;
    uint8_t* ws = (uint8_t*)workspace;
    const int rc = dc_mx4_quantize(x, ws, ws + data, nullptr, nullptr, nullptr, m, k, dtype, 0, nullptr, 0, stream);
    if (rc != DC_OK) return rc;
    return mx4_product(nullptr, ws, ws + data, w_data, w_scales, bias, out, m, n, k, bias_dtype, dtype, (cudaStream_t)stream);
}

// A packed matrix in one piece of memory, the scales behind the codes (both multiples of 16 bytes).
static size_t mx4_bytes(int64_t rows, int64_t cols) { return dc_mx4_data_bytes(rows, cols) + dc_mx4_scale_bytes(rows, cols); }
static uint8_t* mx4_scales_of(void* piece, int64_t rows, int64_t cols) { return piece == nullptr ? nullptr : (uint8_t*)piece + dc_mx4_data_bytes(rows, cols); }
static bool mx4_dtype_ok(int d) { return d >= DC_F32 && d <= DC_BF16; }

size_t dc_mx4_linear_train_workspace_bytes(int64_t m, int64_t n, int64_t k) { return mx4_bytes(m, k) + mx4_bytes(n, k); }

int dc_mx4_linear_train(const void* x, const void* w, const void* bias, void* out, void* xt, void* wt, int64_t m, int64_t n, int64_t k, int32_t dtype,
                        int32_t w_dtype, int32_t bias_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (!mx4_sizes_ok(m, n, k) || m == 0 || n == 0) return DC_ERR_SHAPE;
    if (!mx4_dtype_ok(dtype) || !mx4_dtype_ok(w_dtype) || (bias != nullptr && !mx4_dtype_ok(bias_dtype))) return DC_ERR_DTYPE;
    if (x == nullptr || w == nullptr || out == nullptr || workspace == nullptr) return DC_ERR_NULL_POINTER;
    if (!aligned16(workspace) || !aligned16(xt) || !aligned16(wt)) return DC_ERR_ALIGNMENT;
    if (workspace_bytes < dc_mx4_linear_train_workspace_bytes(m, n, k)) return DC_ERR_WORKSPACE;
    uint8_t *xq = (uint8_t*)workspace, *wq = xq + mx4_bytes(m, k);
    int rc;
    if (xt != nullptr && wt != nullptr && dtype == w_dtype) {
        rc = mx4_quantize_two(x, xq, mx4_scales_of(xq, m, k), xt, mx4_scales_of(xt, k, m), m, w, wq, mx4_scales_of(wq, n, k), wt, mx4_scales_of(wt, k, n), n, k,
                              dtype, (cudaStream_t)stream);
    } else {
        rc = dc_mx4_quantize(x, xq, mx4_scales_of(xq, m, k), xt, mx4_scales_of(xt, k, m), nullptr, m, k, dtype, 0, nullptr, 0, stream);
        if (rc == DC_OK) rc = dc_mx4_quantize(w, wq, mx4_scales_of(wq, n, k), wt, mx4_scales_of(wt, k, n), nullptr, n, k, w_dtype, 0, nullptr, 0, stream);
    }
    if (rc != DC_OK) return rc;
    return mx4_product(nullptr, xq, mx4_scales_of(xq, m, k), wq, mx4_scales_of(wq, n, k), bias, out, m, n, k, bias_dtype, dtype, (cudaStream_t)stream);
}

size_t dc_mx4_linear_backward_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (!mx4_sizes_ok(m, n, k)) return 0;
    return mx4_bytes(m, n) + mx4_bytes(n, m) + dc_mx4_colsum_workspace_bytes(m, n);
}

int dc_mx4_linear_backward(const void* dy, const void* xt, const void* wt, void* dx, void* dw, void* db, int64_t m, int64_t n, int64_t k, int32_t dtype,
                           int32_t w_dtype, int32_t bias_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (!mx4_sizes_ok(m, n, k) || m == 0 || n == 0) return DC_ERR_SHAPE;
    if (!mx4_dtype_ok(dtype) || (dw != nullptr && !mx4_dtype_ok(w_dtype)) || (db != nullptr && !mx4_dtype_ok(bias_dtype))) return DC_ERR_DTYPE;
    if (dx == nullptr && dw == nullptr && db == nullptr) return DC_OK;
    if (dy == nullptr || workspace == nullptr || (dx != nullptr && wt == nullptr) || (dw != nullptr && xt == nullptr)) return DC_ERR_NULL_POINTER;
    if (!aligned16(workspace) || !aligned16(xt) || !aligned16(wt)) return DC_ERR_ALIGNMENT;
    if (workspace_bytes < dc_mx4_linear_backward_workspace_bytes(m, n, k)) return DC_ERR_WORKSPACE;
    uint8_t *dq = (uint8_t*)workspace, *dt = dq + mx4_bytes(m, n), *sums = dt + mx4_bytes(n, m);
    int rc = dc_mx4_quantize(dy, dx != nullptr ? dq : nullptr, dx != nullptr ? mx4_scales_of(dq, m, n) : nullptr, dw != nullptr ? dt : nullptr,
                             dw != nullptr ? mx4_scales_of(dt, n, m) : nullptr, db, m, n, dtype, bias_dtype, db != nullptr ? sums : nullptr,
                             db != nullptr ? dc_mx4_colsum_workspace_bytes(m, n) : 0, stream);
    if (rc == DC_OK && dx != nullptr)
        rc = mx4_product(nullptr, dq, mx4_scales_of(dq, m, n), wt, mx4_scales_of(const_cast<void*>(wt), k, n), nullptr, dx, m, k, n, 0, dtype, (cudaStream_t)stream);
    if (rc == DC_OK && dw != nullptr)
        rc = mx4_product(nullptr, dt, mx4_scales_of(dt, n, m), xt, mx4_scales_of(const_cast<void*>(xt), k, m), nullptr, dw, n, k, m, 0, w_dtype, (cudaStream_t)stream);
    return rc;
}

}  // extern "C"
