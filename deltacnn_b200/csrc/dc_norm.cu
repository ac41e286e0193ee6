// Layer norm over the channel vector of a pixel or token: forward, backward with the column reductions of the weight's
// and bias's gradients, and the delta form with its caches.
//
// Mathematics: mean m = sum x / C, variance v = sum (x - m)^2 / C (two sums over values held in registers: no
// cancellation between large sums), r = 1 / sqrt(v + eps), n = (x - m) r, y = n w + b. Backward, with g = dy w:
// dx = r (g - mean(g) - n mean(g n)), dw = sum_rows dy n, db = sum_rows dy.
//
// Split: a row belongs to a team of threads that keeps it in registers between its one read and its one write: an aligned
// group of lanes while the row has at most 128 packs of 16 bytes (backward: 64; several short rows share a warp, sums are
// shuffles), a whole CTA above that. Teams walk rows with the grid's stride and have the next rows on their way (cp.async into
// their own slots of shared memory); weight, and the column sums of the backward pass, stay in registers, whose per-CTA rests a
// second kernel adds in a fixed order. Rows whose width or address does not allow 16-byte accesses take the same code with
// two halves or single elements (delta form, 82 channels 73 x 18 x 42: 44 us with single halves, 18 with two); rows beyond the
// registers of a CTA pass through shared memory (forward) or are read twice (backward).
//
// Bound: memory, once the arithmetic is packed (two float32 per instruction): 16384 x 4096 bf16 forward 45 us (268 MB, 41 us at
// the copy rate), backward 72 us (403 MB, 61 us); with scalar arithmetic and a branch per pack the issue slots were the bound
// (58 and 99 us). 12544 x 576 fp16 forward 9 us (29 MB, 4.4 us: launch and two round trips). Delta form, fp16: 64 channels
// 136 x 240 x 32, a tenth active, 25 us (83 MB, 12.7 us: sparse pixels leave teams idle); 96 channels 56 x 56 x 64, all active, 43 us
// (231 MB, 35 us). Without 16-byte accesses the issue slots and the reads in flight bound it: 11181 x 3001 bf16 forward 46 us, backward
// 71 us (20 and 31 at the copy rate), 6211 x 5402 28 and 79 us, fp32 11181 x 3001 49 and 87 us (41 and 61).
#include <initializer_list>
#include <type_traits>
#include "dc_common.cuh"

namespace dc {

// W consecutive elements in storage precision: 16-byte accesses, one of 8 or 4 bytes, or an element.
template <typename T, int W> struct Frag {
    static constexpr int kBytes = W * (int)sizeof(T);
    alignas(kBytes % 16 == 0 ? 16 : kBytes) T s[W];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kBytes % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(s)[i] = reinterpret_cast<const uint4*>(p)[i];
        } else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(s) = *reinterpret_cast<const uint2*>(p);
        else if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(s) = *reinterpret_cast<const uint32_t*>(p);
        else s[0] = p[0];
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kBytes % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(s)[i];
        } else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(s);
        else if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(s);
        else p[0] = s[0];
    }
    __device__ __forceinline__ float get(int i) const { return to_f<T>(s[i]); }
    __device__ __forceinline__ void set(int i, float x) { s[i] = from_f<T>(x); }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int i = 0; i < W; ++i) set(i, x);
    }
};

// Float32 values in twos (packed instructions, half the issue slots) for 16-byte packs, singly for single elements.
struct V2 {
    uint64_t v;
    static __device__ __forceinline__ V2 make(float a, float b) { V2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b)); return r; }
    static __device__ __forceinline__ V2 all(float a) { return make(a, a); }
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
    __device__ __forceinline__ float sum() const { float a, b; get(a, b); return a + b; }
};
__device__ __forceinline__ V2 add(V2 a, V2 b) { V2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ V2 mul(V2 a, V2 b) { V2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ V2 fma(V2 a, V2 b, V2 c) { V2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
struct V1 {
    float v;
    static __device__ __forceinline__ V1 all(float a) { return V1{a}; }
    __device__ __forceinline__ float sum() const { return v; }
};
__device__ __forceinline__ V1 add(V1 a, V1 b) { return V1{a.v + b.v}; }
__device__ __forceinline__ V1 mul(V1 a, V1 b) { return V1{a.v * b.v}; }
__device__ __forceinline__ V1 fma(V1 a, V1 b, V1 c) { return V1{fmaf(a.v, b.v, c.v)}; }

// The values of a Frag in float32.
template <int W> struct Vals {
    using V = V2;
    static constexpr int N = W / 2;
    V2 v[N];
    template <typename T> __device__ __forceinline__ void from(const Frag<T, W>& f) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = V2::make(f.s[2 * i], f.s[2 * i + 1]);
            else if constexpr (std::is_same_v<T, __half>) {
                const float2 h = __half22float2(reinterpret_cast<const __half2*>(f.s)[i]);
                v[i] = V2::make(h.x, h.y);
            } else {
                const uint32_t u = reinterpret_cast<const uint32_t*>(f.s)[i];
                v[i] = V2::make(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
            }
        }
    }
    template <typename T> __device__ __forceinline__ void to(Frag<T, W>& f) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float a, b;
            v[i].get(a, b);
            if constexpr (sizeof(T) == 4) { f.s[2 * i] = a; f.s[2 * i + 1] = b; }
            else if constexpr (std::is_same_v<T, __half>) reinterpret_cast<__half2*>(f.s)[i] = __floats2half2_rn(a, b);
            else reinterpret_cast<__nv_bfloat162*>(f.s)[i] = __floats2bfloat162_rn(a, b);
        }
    }
    __device__ __forceinline__ void put(float* p) const {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i].get(p[2 * i], p[2 * i + 1]);
    }
};
template <> struct Vals<1> {
    using V = V1;
    static constexpr int N = 1;
    V1 v[1];
    template <typename T> __device__ __forceinline__ void from(const Frag<T, 1>& f) { v[0].v = to_f<T>(f.s[0]); }
    template <typename T> __device__ __forceinline__ void to(Frag<T, 1>& f) const { f.s[0] = from_f<T>(v[0].v); }
    __device__ __forceinline__ void put(float* p) const { p[0] = v[0].v; }
};

constexpr int kLnCta = 512;         // most threads of a CTA that holds a row: 128 registers a thread
// Threads of a CTA at most for a row split into so many packs per thread.
__host__ __device__ constexpr int row_threads(int w, int p) { return (w <= 2 ? p > 4 : p > 1) ? kLnCta : 256; }
constexpr int kMaxWarps = 32;

// Sum over an aligned group of g lanes, g the same in the whole grid: five predicated steps instead of a loop.
__device__ __forceinline__ float lanes_sum(float x, int g) {
    if (g > 16) x += __shfl_xor_sync(DC_FULL, x, 16);
    if (g > 8) x += __shfl_xor_sync(DC_FULL, x, 8);
    if (g > 4) x += __shfl_xor_sync(DC_FULL, x, 4);
    if (g > 2) x += __shfl_xor_sync(DC_FULL, x, 2);
    if (g > 1) x += __shfl_xor_sync(DC_FULL, x, 1);
    return x;
}

// A row's team: g lanes of a warp (BLOCK false) or the whole CTA (BLOCK true).
// Pack k of a thread is first + k hop(): the lanes of a group go round; in a CTA every warp has a stretch of 32 P packs of its own,
// so that a thread's packs are one address with constant offsets and only the last warps look where the row ends.
template <bool BLOCK, int P = 1> struct Team {
    int rank, size;            // this thread's place in the team, the team's threads
    int first;
    int64_t row, stride;       // first row, distance to the next one
    __device__ __forceinline__ Team(int g) {
        if constexpr (BLOCK) {
            rank = threadIdx.x; size = blockDim.x; row = blockIdx.x; stride = gridDim.x;
            first = (threadIdx.x >> 5) * 32 * P + (threadIdx.x & 31);
        } else {
            const int per_cta = blockDim.x / g;
            rank = first = threadIdx.x & (g - 1); size = g;
            row = (int64_t)blockIdx.x * per_cta + threadIdx.x / g;
            stride = (int64_t)gridDim.x * per_cta;
        }
    }
    __device__ __forceinline__ int hop() const { return BLOCK ? 32 : size; }
    // Sum over the team, the same bits in every thread. red: kMaxWarps floats per call site (BLOCK); a site is used again
    // only after another site's barrier.
    __device__ __forceinline__ float sum(float x, float* red) const {
        if constexpr (!BLOCK) return lanes_sum(x, size);
        x = group_sum(x, 32);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
        __syncthreads();
        const int lane = threadIdx.x & 31;
        return group_sum(lane < (int)(blockDim.x >> 5) ? red[lane] : 0.f, 32);
    }
};

// f(k, pack k is inside the row) for a thread's packs. SPLIT: warps that are inside as a whole (`all`) run it without the question.
template <int P, bool SPLIT, typename F> __device__ __forceinline__ void each_pack(bool all, unsigned valid, F&& f) {
    if (SPLIT && all) {
#pragma unroll
        for (int k = 0; k < P; ++k) f(k, true);
    } else {
#pragma unroll
        for (int k = 0; k < P; ++k) f(k, (valid >> k & 1u) != 0);
    }
}

// The rows ahead of the one at hand. 16-byte packs: every thread copies its own packs of the next rows of N arrays into its own
// slots of a ring in shared memory (cp.async: no registers, no barrier, a wait for the thread's own copies). Three rows, or one
// where a row alone is 64 KB or more of a CTA's shared memory. Single elements: the next row in registers.
__host__ __device__ constexpr int rows_ahead(int packs) { return packs > 4 ? 1 : 3; }
__device__ __forceinline__ void cp16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
// Packs behind the end of a row (rank + k size >= nvec) read as zeros, so that the arithmetic needs no branch for them.
template <typename T, int W, int P, int N, bool BLOCK> struct RowPipe {
    static constexpr bool kRing = W * sizeof(T) == 16;
    static constexpr int kAhead = rows_ahead(N * P);
    Frag<T, W> next[kRing ? 1 : N][kRing ? 1 : P];
    uint8_t* mine;
    const T* at[N];                        // this thread's first pack of the next row to ask for
    int64_t step, left;                    // elements between the team's rows; rows it still has to ask for
    int group, in, out;                    // slots to fill, to read
    unsigned valid;                        // bit k: pack k is inside the row
    bool all;                              // all packs of the warp are
    __device__ __forceinline__ int hop() const { return BLOCK ? 32 : group; }
    template <typename F> __device__ __forceinline__ void each(F&& f) const { each_pack<P, BLOCK && !kRing>(all, valid, f); }

    __device__ __forceinline__ void ask() {
        if (left > 0) {
            each([&](int k, bool inside) {
                if (!inside) return;
#pragma unroll
                for (int n = 0; n < N; ++n)
                    if constexpr (kRing) cp16(mine + (size_t)((in * N + n) * P + k) * blockDim.x * 16, at[n] + k * hop() * W);
                    else next[n][k].load(at[n] + k * hop() * W);
            });
#pragma unroll
            for (int n = 0; n < N; ++n) at[n] += step;
        }
        if constexpr (kRing) {
            asm volatile("cp.async.commit_group;" ::: "memory");
            in = in == kAhead ? 0 : in + 1;
        }
        --left;
    }
    __device__ __forceinline__ void start(const Team<BLOCK, P>& t, const void* const (&src)[N], int64_t rows, int c, int nvec, uint8_t* smem) {
        mine = smem + threadIdx.x * 16;
        group = t.size;
        step = t.stride * c;
        left = t.row < rows ? (rows - t.row + t.stride - 1) / t.stride : 0;
        in = out = 0;
        valid = 0;
#pragma unroll
        for (int k = 0; k < P; ++k) valid |= t.first + k * t.hop() < nvec ? 1u << k : 0u;
        all = __all_sync(DC_FULL, valid == (1u << P) - 1u);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            at[n] = (const T*)src[n] + t.row * c + t.first * W;
#pragma unroll
            for (int k = 0; k < P; ++k) {
                if constexpr (kRing) {
                    if (!(valid >> k & 1u))
                        for (int i = 0; i <= kAhead; ++i)
                            *reinterpret_cast<uint4*>(mine + (size_t)((i * N + n) * P + k) * blockDim.x * 16) = make_uint4(0u, 0u, 0u, 0u);
                } else {
                    next[n][k].fill(0.f);
                }
            }
        }
        for (int i = 0; i < (kRing ? kAhead : 1); ++i) ask();
    }
    // The current row's packs, with the next request on its way.
    __device__ __forceinline__ void take(Frag<T, W> (&v)[N][P]) {
        if constexpr (kRing) {
            ask();
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < P; ++k) v[n][k].load(reinterpret_cast<const T*>(mine + (size_t)((out * N + n) * P + k) * blockDim.x * 16));
            out = out == kAhead ? 0 : out + 1;
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < P; ++k) v[n][k] = next[n][k];
            ask();
        }
    }
};

template <typename T, int W, int P>
__device__ __forceinline__ void load_param(Frag<T, W> (&v)[P], const T* p, int rank, int size, int nvec, float neutral) {
#pragma unroll
    for (int k = 0; k < P; ++k) {
        v[k].fill(rank + k * size < nvec ? neutral : 0.f);
        if (p != nullptr && rank + k * size < nvec) v[k].load(p + (rank + k * size) * W);
    }
}

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------
struct LnParams {
    const void *x, *w, *b;
    void* y;
    float *mean, *rstd;
    int64_t rows;
    int c, nvec, g;
    float eps, inv_c;
};

template <typename T, typename WT, int W, int P, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? row_threads(W, P) : 256) k_ln_fwd(LnParams p) {
    __shared__ float red[2][kMaxWarps];
    extern __shared__ __align__(16) uint8_t ring[];
    grid_dep_launch();
    grid_dep_wait();
    const Team<BLOCK, P> t(p.g);
    RowPipe<T, W, P, 1, BLOCK> pipe;
    pipe.start(t, {p.x}, p.rows, p.c, p.nvec, ring);
    T* y = (T*)p.y + t.row * p.c + t.first * W;
    // weight and bias stay in registers; lanes with three packs and more read them from L1 for every row instead and have the
    // registers for twice the warps (12544 x 576: 12.3 -> 8.9 us)
    constexpr bool kHeld = BLOCK || P < 3 || W <= 2;
    Frag<WT, W> w[kHeld ? P : 1], b[kHeld ? P : 1];
    if constexpr (kHeld) {
        load_param<WT, W, P>(w, (const WT*)p.w, t.first, t.hop(), p.nvec, 1.f);
        load_param<WT, W, P>(b, (const WT*)p.b, t.first, t.hop(), p.nvec, 0.f);
    }
    using V = typename Vals<W>::V;
    constexpr int N = Vals<W>::N;
    // lanes of a warp whose own rows have run out still take part in its shuffles
    for (int64_t base = t.row - (BLOCK ? 0 : (threadIdx.x & 31) / p.g), row = t.row; base < p.rows; base += t.stride, row += t.stride, y += pipe.step) {
        const bool on = BLOCK || row < p.rows;
        Frag<T, W> in[1][P];
        pipe.take(in);
        Vals<W> x[P];
        V s = V::all(0.f), q = V::all(0.f);
#pragma unroll
        for (int k = 0; k < P; ++k) {
            x[k].from(in[0][k]);
#pragma unroll
            for (int i = 0; i < N; ++i) s = add(s, x[k].v[i]);
        }
        const float m = t.sum(s.sum(), red[0]) * p.inv_c;
        pipe.each([&](int k, bool inside) {
            const V neg = V::all(inside ? -m : 0.f);
#pragma unroll
            for (int i = 0; i < N; ++i) { x[k].v[i] = add(x[k].v[i], neg); q = fma(x[k].v[i], x[k].v[i], q); }
        });
        const float r = rsqrtf(t.sum(q.sum(), red[1]) * p.inv_c + p.eps);
        const V rr = V::all(r);
        pipe.each([&](int k, bool inside) {
            Vals<W> ww, bb;
            if constexpr (kHeld) {
                ww.from(w[k]);
                bb.from(b[k]);
            } else {
                Frag<WT, W> f[2];
                f[0].fill(1.f);
                f[1].fill(0.f);
                const int col = (t.first + k * t.hop()) * W;
                if (p.w != nullptr && inside) f[0].load((const WT*)p.w + col);
                if (p.b != nullptr && inside) f[1].load((const WT*)p.b + col);
                ww.from(f[0]);
                bb.from(f[1]);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) x[k].v[i] = fma(mul(x[k].v[i], rr), ww.v[i], bb.v[i]);
            x[k].to(in[0][k]);
            if (on && inside) in[0][k].store(y + k * t.hop() * W);
        });
        if (on && t.rank == 0 && p.mean != nullptr) { p.mean[row] = m; p.rstd[row] = r; }
    }
}

// Rows beyond the registers of a CTA. Three CTAs of 512 threads per SM, so that one's barriers pass under another's reads; every
// thread asks for several packs before it uses the first.
constexpr int kLongThreads = 512, kLongCtas = 3;
template <int W> constexpr int kLongBatch = W == 1 ? 8 : W == 8 ? 1 : W == 2 ? 4 : 2;
constexpr int kLongSmem = 200 * 1024;

// A thread's packs of a row of n, a batch at a time: body(first pack, all of them inside the row). The CTA's size is a constant,
// so that a batch's accesses are one address with constant offsets, and only the last batch looks where the row ends: with a
// bound on every element and 64-bit products for its address a forward pass of 15001 elements in bf16 took 79 instructions per
// element, and 104 us instead of 58 us for 2236 rows.
template <int W, typename F>
__device__ __forceinline__ void long_row(int n, F&& body) {
    constexpr int B = kLongBatch<W>;
    int i = threadIdx.x;
    for (; i + (B - 1) * kLongThreads < n; i += B * kLongThreads) body(i, std::true_type{});
    if (i < n) body(i, std::false_type{});
}
// Packs i, i + kLongThreads, ... of p; those behind the end, and all of an absent one, are `other`.
template <bool ALL, typename T, int W>
__device__ __forceinline__ void long_load(Frag<T, W> (&v)[kLongBatch<W>], const T* p, int i, int n, float other) {
    p += (int64_t)i * W;
#pragma unroll
    for (int k = 0; k < kLongBatch<W>; ++k)
        if (ALL || i + k * kLongThreads < n) v[k].load(p + k * kLongThreads * W);
        else v[k].fill(other);
}
template <bool ALL, typename T, int W>
__device__ __forceinline__ void long_param(Frag<T, W> (&v)[kLongBatch<W>], const T* p, int i, int n, float other) {
    if (p != nullptr) long_load<ALL, T, W>(v, p, i, n, other);
    else
#pragma unroll
        for (int k = 0; k < kLongBatch<W>; ++k) v[k].fill(other);
}

// One read of a row that shared memory holds meanwhile (HELD: every thread reads back its own packs); longer ones are read three
// times, the second and third time mostly from L2.
template <typename T, typename WT, int W, bool HELD>
__global__ void __launch_bounds__(kLongThreads, kLongCtas) k_ln_fwd_long(LnParams p) {
    __shared__ float red[2][kMaxWarps];
    extern __shared__ __align__(16) uint8_t held[];
    constexpr int B = kLongBatch<W>;
    using V = typename Vals<W>::V;
    constexpr int N = Vals<W>::N;
    grid_dep_launch();
    grid_dep_wait();
    const Team<true> t(0);
    for (int64_t row = t.row; row < p.rows; row += t.stride) {
        const T* x = (const T*)p.x + row * p.c;
        const T* again = HELD ? reinterpret_cast<const T*>(held) : x;
        T* y = (T*)p.y + row * p.c;
        V s = V::all(0.f), q = V::all(0.f);
        long_row<W>(p.nvec, [&](int i, auto all) {
            Frag<T, W> v[B];
            long_load<all.value, T, W>(v, x, i, p.nvec, 0.f);
#pragma unroll
            for (int k = 0; k < B; ++k) {
                if (HELD && (all.value || i + k * kLongThreads < p.nvec)) v[k].store(reinterpret_cast<T*>(held) + (i + k * kLongThreads) * W);
                Vals<W> f;
                f.from(v[k]);
#pragma unroll
                for (int j = 0; j < N; ++j) s = add(s, f.v[j]);
            }
        });
        const float m = t.sum(s.sum(), red[0]) * p.inv_c;
        const V neg = V::all(-m);
        long_row<W>(p.nvec, [&](int i, auto all) {
            Frag<T, W> v[B];
            long_load<all.value, T, W>(v, again, i, p.nvec, 0.f);
#pragma unroll
            for (int k = 0; k < B; ++k)
                if (all.value || i + k * kLongThreads < p.nvec) {
                    Vals<W> f;
                    f.from(v[k]);
#pragma unroll
                    for (int j = 0; j < N; ++j) { const V d = add(f.v[j], neg); q = fma(d, d, q); }
                }
        });
        const float r = rsqrtf(t.sum(q.sum(), red[1]) * p.inv_c + p.eps);
        const V rr = V::all(r);
        long_row<W>(p.nvec, [&](int i, auto all) {
            Frag<T, W> v[B];
            Frag<WT, W> w[B], b[B];
            long_load<all.value, T, W>(v, again, i, p.nvec, 0.f);
            long_param<all.value, WT, W>(w, (const WT*)p.w, i, p.nvec, 1.f);
            long_param<all.value, WT, W>(b, (const WT*)p.b, i, p.nvec, 0.f);
            T* const o = y + (int64_t)i * W;
#pragma unroll
            for (int k = 0; k < B; ++k) {
                Vals<W> f, ww, bb;
                f.from(v[k]);
                ww.from(w[k]);
                bb.from(b[k]);
#pragma unroll
                for (int j = 0; j < N; ++j) f.v[j] = fma(mul(add(f.v[j], neg), rr), ww.v[j], bb.v[j]);
                f.to(v[k]);
                if (all.value || i + k * kLongThreads < p.nvec) v[k].store(o + k * kLongThreads * W);
            }
        });
        if (t.rank == 0 && p.mean != nullptr) { p.mean[row] = m; p.rstd[row] = r; }
    }
}

// ---------------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------------
struct LnBwdParams {
    const void *dy, *x, *w;
    const float *mean, *rstd;
    void* dx;
    float* partial;            // [slices][2][c]: a CTA's sums of dy n and dy; NULL: not wanted
    float* means;              // long rows: [rows][2], the rows' means of g and g n
    int64_t rows, per;         // per: long rows, rows of a block
    int c, nvec, g;
    float inv_c;
};

// CTAs of so many threads whose registers an SM holds: the accumulators alone are 2 P W registers.
__host__ __device__ constexpr int bwd_ctas(int w, int p) { return row_threads(w, p) == kLnCta ? 1 : w == 2 && p > 2 ? 2 : 3; }

template <typename T, typename WT, int W, int P, bool BLOCK>
__global__ void __launch_bounds__(row_threads(W, P), bwd_ctas(W, P)) k_ln_bwd(LnBwdParams p) {
    __shared__ float red[2][2][kMaxWarps];
    extern __shared__ __align__(16) uint8_t ring[];      // the rows ahead; at the end [2][c] column sums of the CTA's teams
    grid_dep_launch();
    grid_dep_wait();
    const Team<BLOCK, P> t(p.g);
    RowPipe<T, W, P, 2, BLOCK> pipe;
    pipe.start(t, {p.x, p.dy}, p.rows, p.c, p.nvec, ring);
    T* dx = (T*)p.dx + t.row * p.c + t.first * W;
    Frag<WT, W> w[P];
    load_param<WT, W, P>(w, (const WT*)p.w, t.first, t.hop(), p.nvec, 1.f);
    using V = typename Vals<W>::V;
    constexpr int N = Vals<W>::N;
    Vals<W> dw[P], db[P];
#pragma unroll
    for (int k = 0; k < P; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) dw[k].v[i] = db[k].v[i] = V::all(0.f);
    float nm = 0.f, nr = 0.f;
    [[maybe_unused]] int par = 0;
    if (t.row < p.rows) { nm = p.mean[t.row]; nr = p.rstd[t.row]; }
    for (int64_t base = t.row - (BLOCK ? 0 : (threadIdx.x & 31) / p.g), row = t.row; base < p.rows; base += t.stride, row += t.stride, dx += pipe.step) {
        const bool on = BLOCK || row < p.rows;
        const float m = nm, r = nr;
        Frag<T, W> in[2][P];
        pipe.take(in);
        if (row + t.stride < p.rows) { nm = p.mean[row + t.stride]; nr = p.rstd[row + t.stride]; }
        // n and g stay in registers between the two sums and dx, or are formed again where a thread has too many of them
        constexpr bool kKeep = P * W <= 16 && P < 16;
        Vals<W> n[kKeep ? P : 1], g[kKeep ? P : 1];
        V sg = V::all(0.f), sgn = V::all(0.f);
        const V rr = V::all(r);
        auto form = [&](int k, bool inside, Vals<W>& nn, Vals<W>& ee, Vals<W>& gg) {
            Vals<W> ww;
            nn.from(in[0][k]);
            ee.from(in[1][k]);
            ww.from(w[k]);
            const V shift = V::all(inside ? -m : 0.f);
#pragma unroll
            for (int i = 0; i < N; ++i) { nn.v[i] = mul(add(nn.v[i], shift), rr); gg.v[i] = mul(ee.v[i], ww.v[i]); }
        };
        if (on)
            pipe.each([&](int k, bool inside) {
                Vals<W> nn, ee, gg;
                form(k, inside, nn, ee, gg);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    dw[k].v[i] = fma(ee.v[i], nn.v[i], dw[k].v[i]);
                    db[k].v[i] = add(db[k].v[i], ee.v[i]);
                    sg = add(sg, gg.v[i]);
                    sgn = fma(gg.v[i], nn.v[i], sgn);
                }
                if constexpr (kKeep) { n[k] = nn; g[k] = gg; }
            });
        if (p.dx != nullptr) {
            float a, c;
            if constexpr (BLOCK) {             // both sums behind one barrier
                const int lane = threadIdx.x & 31;
                par ^= 1;
                a = group_sum(sg.sum(), 32);
                c = group_sum(sgn.sum(), 32);
                if (lane == 0) { red[par][0][threadIdx.x >> 5] = a; red[par][1][threadIdx.x >> 5] = c; }
                __syncthreads();
                const bool in_cta = lane < (int)(blockDim.x >> 5);
                a = group_sum(in_cta ? red[par][0][lane] : 0.f, 32) * p.inv_c;
                c = group_sum(in_cta ? red[par][1][lane] : 0.f, 32) * p.inv_c;
            } else {
                a = lanes_sum(sg.sum(), t.size) * p.inv_c;
                c = lanes_sum(sgn.sum(), t.size) * p.inv_c;
            }
            const V na = V::all(-a), nc = V::all(-c);
            pipe.each([&](int k, bool inside) {
                Vals<W> nn, ee, gg;
                if constexpr (kKeep) { nn = n[k]; gg = g[k]; }
                else form(k, inside, nn, ee, gg);
#pragma unroll
                for (int i = 0; i < N; ++i) gg.v[i] = mul(rr, fma(nn.v[i], nc, add(gg.v[i], na)));
                gg.to(in[0][k]);
                if (on && inside) in[0][k].store(dx + k * t.hop() * W);
            });
        }
    }
    if (p.partial == nullptr) return;
    float* out = p.partial + (int64_t)blockIdx.x * 2 * p.c;
    if constexpr (BLOCK) {
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (t.first + k * t.hop() < p.nvec) {
                const int col = (t.first + k * t.hop()) * W;
                Frag<float, W> f;
                dw[k].put(f.s);
                f.store(out + col);
                db[k].put(f.s);
                f.store(out + p.c + col);
            }
    } else {
        // teams of a warp by shuffles, warps of the CTA one after the other: a fixed order
        float* cols = reinterpret_cast<float*>(ring);
        __syncthreads();                       // every thread has read its last row
        float sums[2][P][W];
#pragma unroll
        for (int k = 0; k < P; ++k) {
            dw[k].put(sums[0][k]);
            db[k].put(sums[1][k]);
#pragma unroll
            for (int i = 0; i < W; ++i)
                for (int o = p.g; o < 32; o <<= 1) {
                    sums[0][k][i] += __shfl_xor_sync(DC_FULL, sums[0][k][i], o);
                    sums[1][k][i] += __shfl_xor_sync(DC_FULL, sums[1][k][i], o);
                }
        }
        const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        for (int q = 0; q < warps; ++q) {
            if (warp == q && (threadIdx.x & 31) < p.g) {
#pragma unroll
                for (int k = 0; k < P; ++k)
                    if (t.first + k * t.hop() < p.nvec)
#pragma unroll
                        for (int i = 0; i < W; ++i) {
                            const int col = (t.first + k * t.hop()) * W + i;
                            cols[col] = (q == 0 ? 0.f : cols[col]) + sums[0][k][i];
                            cols[p.c + col] = (q == 0 ? 0.f : cols[p.c + col]) + sums[1][k][i];
                        }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 2 * p.c; i += blockDim.x) out[i] = cols[i];
    }
}

// Long rows, in two kernels (2236 x 15001 in bf16 227 -> 132 us, 1677 x 20000 205 -> 67 us against one that kept the column sums in
// shared memory), since no thread can keep the column sums of a whole row's share: the rows' two means (every row once),
// then dx and the column sums by CTAs that own a block of columns and walk down some rows (every row once more, and weight and
// the sums in registers). The second read comes from L2 where the batch fits there.
template <typename T, typename WT, int W>
__global__ void __launch_bounds__(kLongThreads, kLongCtas) k_ln_bwd_means(LnBwdParams p) {
    __shared__ float red[2][kMaxWarps];
    constexpr int B = kLongBatch<W>;
    using V = typename Vals<W>::V;
    constexpr int N = Vals<W>::N;
    grid_dep_launch();
    grid_dep_wait();
    const Team<true> t(0);
    for (int64_t row = t.row; row < p.rows; row += t.stride) {
        const T *x = (const T*)p.x + row * p.c, *dy = (const T*)p.dy + row * p.c;
        const V neg = V::all(-p.mean[row]), r = V::all(p.rstd[row]);
        V sg = V::all(0.f), sgn = V::all(0.f);
        long_row<W>(p.nvec, [&](int i, auto all) {
            Frag<T, W> v[B], d[B];
            Frag<WT, W> w[B];
            long_load<all.value, T, W>(v, x, i, p.nvec, 0.f);
            long_load<all.value, T, W>(d, dy, i, p.nvec, 0.f);
            long_param<all.value, WT, W>(w, (const WT*)p.w, i, p.nvec, 1.f);
#pragma unroll
            for (int k = 0; k < B; ++k)
                if (all.value || i + k * kLongThreads < p.nvec) {
                    Vals<W> n, e, ww;
                    n.from(v[k]);
                    e.from(d[k]);
                    ww.from(w[k]);
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const V g = mul(e.v[j], ww.v[j]);
                        sg = add(sg, g);
                        sgn = fma(g, mul(add(n.v[j], neg), r), sgn);
                    }
                }
        });
        const float a = t.sum(sg.sum(), red[0]) * p.inv_c, c = t.sum(sgn.sum(), red[1]) * p.inv_c;
        if (t.rank == 0) { p.means[2 * row] = a; p.means[2 * row + 1] = c; }
    }
}

constexpr int kColThreads = 256, kColCtas = 3, kColMinRows = 8;
template <int W> constexpr int kColRows = W == 8 ? 2 : 4;      // in flight
template <int W> constexpr int kColPacks = W >= 4 ? 1 : 4 / W;
// grid: blocks of columns x blocks of p.per rows.
template <typename T, typename WT, int W>
__global__ void __launch_bounds__(kColThreads, kColCtas) k_ln_bwd_cols(LnBwdParams p) {
    constexpr int K = kColPacks<W>, R = kColRows<W>;
    using V = typename Vals<W>::V;
    constexpr int N = Vals<W>::N;
    grid_dep_launch();
    grid_dep_wait();
    const int first = blockIdx.x * kColThreads * K + threadIdx.x;
    Frag<WT, W> w[K];
    load_param<WT, W, K>(w, (const WT*)p.w, first, kColThreads, p.nvec, 1.f);
    Vals<W> dw[K], db[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) dw[k].v[i] = db[k].v[i] = V::all(0.f);
    const int64_t begin = (int64_t)blockIdx.y * p.per, end = begin + p.per < p.rows ? begin + p.per : p.rows;
    unsigned valid = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) valid |= first + k * kColThreads < p.nvec ? 1u << k : 0u;
    int64_t at = begin * p.c + (int64_t)first * W;
    // rows row ... row + R - 1; ALL: none is behind the end, and all of the thread's columns are inside
    auto take = [&](int64_t row, auto all) {
        constexpr bool ALL = all.value;
        Frag<T, W> x[R][K], dy[R][K];
        float m[R], r[R], a[R], c[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const bool on = ALL || row + j < end;
            m[j] = r[j] = a[j] = c[j] = 0.f;
            if (on) {
                m[j] = p.mean[row + j];
                r[j] = p.rstd[row + j];
                if (p.dx != nullptr) { a[j] = p.means[2 * (row + j)]; c[j] = p.means[2 * (row + j) + 1]; }
            }
            const T *px = (const T*)p.x + at + (int64_t)j * p.c, *pd = (const T*)p.dy + at + (int64_t)j * p.c;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (ALL || (on && (valid >> k & 1u))) {
                    x[j][k].load(px + k * kColThreads * W);
                    dy[j][k].load(pd + k * kColThreads * W);
                } else {
                    x[j][k].fill(0.f);
                    dy[j][k].fill(0.f);
                }
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const V neg = V::all(-m[j]), rr = V::all(r[j]), na = V::all(-a[j]), nc = V::all(-c[j]);
            T* o = (T*)p.dx + at + (int64_t)j * p.c;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                Vals<W> n, e, ww;
                n.from(x[j][k]);
                e.from(dy[j][k]);
                ww.from(w[k]);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    n.v[i] = mul(add(n.v[i], neg), rr);
                    dw[k].v[i] = fma(e.v[i], n.v[i], dw[k].v[i]);
                    db[k].v[i] = add(db[k].v[i], e.v[i]);
                    e.v[i] = mul(rr, fma(n.v[i], nc, add(mul(e.v[i], ww.v[i]), na)));
                }
                if (p.dx != nullptr && (ALL || (row + j < end && (valid >> k & 1u)))) {
                    e.to(x[j][k]);
                    x[j][k].store(o + k * kColThreads * W);
                }
            }
        }
    };
    int64_t row = begin;
    if (valid == (1u << K) - 1)
        for (; row + R <= end; row += R, at += (int64_t)R * p.c) take(row, std::true_type{});
    for (; row < end; row += R, at += (int64_t)R * p.c) take(row, std::false_type{});
    if (p.partial == nullptr) return;
    float* out = p.partial + (int64_t)blockIdx.y * 2 * p.c;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (first + k * kColThreads < p.nvec) {
            const int col = (first + k * kColThreads) * W;
            Frag<float, W> f;
            dw[k].put(f.s);
            f.store(out + col);
            db[k].put(f.s);
            f.store(out + p.c + col);
        }
}

// Column sums of the CTAs' partial rows, in a fixed order: 32 columns per CTA, R threads share a column's rows and have four of
// them in flight each. R = 32; 4 for few rows, where the threads of a wide CTA would find nothing (4 rows of 14801 columns: 14
// -> 10 us, started under the kernel before; with 16 threads and one row at a time 296 rows of 4096 took 17 us, all latency).
template <typename OT, int R>
__global__ void __launch_bounds__(32 * R) k_col_reduce(const float* __restrict__ partial, int n, int c, int64_t pitch, OT* __restrict__ o0,
                                                       OT* __restrict__ o1) {
    __shared__ float s[R][33];
    grid_dep_launch();
    grid_dep_wait();
    const int col = blockIdx.x * 32 + threadIdx.x;
    OT* o = blockIdx.y == 0 ? o0 : o1;
    if (o == nullptr) return;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (col < c) {
        const float* src = partial + (int64_t)blockIdx.y * c + col;
        for (int i = threadIdx.y; i < n; i += 4 * R) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j * R < n) a[j] += src[(i + j * R) * pitch];
        }
    }
    s[threadIdx.y][threadIdx.x] = (a[0] + a[1]) + (a[2] + a[3]);
    __syncthreads();
    if (threadIdx.y == 0 && col < c) {
        float v[4] = {s[0][threadIdx.x], s[1][threadIdx.x], s[2][threadIdx.x], s[3][threadIdx.x]};
#pragma unroll
        for (int i = 4; i < R; ++i) v[i & 3] += s[i][threadIdx.x];
        o[col] = from_f<OT>((v[0] + v[1]) + (v[2] + v[3]));
    }
}

template <typename OT>
static int col_reduce_t(const float* partial, int n, int c, int64_t pitch, void* o0, void* o1, cudaStream_t st) {
    const dim3 grid((unsigned)divup(c, 32), o1 != nullptr ? 2u : 1u);
    if (n <= 64) return launch_pdl(k_col_reduce<OT, 4>, grid, dim3(32, 4), 0, st, partial, n, c, pitch, (OT*)o0, (OT*)o1);
    return launch_pdl(k_col_reduce<OT, 32>, grid, dim3(32, 32), 0, st, partial, n, c, pitch, (OT*)o0, (OT*)o1);
}
int col_reduce(const float* partial, int n, int c, int64_t pitch, void* o0, void* o1, int dtype, cudaStream_t st) {
    switch (dtype) {
        case DC_F32: return col_reduce_t<float>(partial, n, c, pitch, o0, o1, st);
        case DC_F16: return col_reduce_t<__half>(partial, n, c, pitch, o0, o1, st);
        case DC_BF16: return col_reduce_t<__nv_bfloat16>(partial, n, c, pitch, o0, o1, st);
        default: return DC_ERR_DTYPE;
    }
}

// ---------------------------------------------------------------------------------------------
// delta form
// ---------------------------------------------------------------------------------------------
struct LnDeltaParams {
    const void *delta, *w, *b;
    const int32_t* mask;
    void *prev_in, *prev_out, *out;
    int32_t* mask_out;
    int64_t npix;
    int c, nvec, g;
    float thr, eps, inv_c;
    int chunk;                 // pixels that a warp takes at once (teams of lanes)
};

// Sums and differences in the storage type, each rounded once. Two halves added in packed half arithmetic give the correctly
// rounded half, as float32 and one rounding do (24 >= 2 * 11 + 2 bits).
template <typename T, int W> __device__ __forceinline__ void frag_add(Frag<T, W>& a, const Frag<T, W>& b) {
    if constexpr (std::is_same_v<T, __half> && W > 1) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) reinterpret_cast<__half2*>(a.s)[i] = __hadd2(reinterpret_cast<__half2*>(a.s)[i], reinterpret_cast<const __half2*>(b.s)[i]);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) a.set(i, a.get(i) + b.get(i));
    }
}
template <typename T, int W> __device__ __forceinline__ void frag_sub(Frag<T, W>& a, const Frag<T, W>& b) {
    if constexpr (std::is_same_v<T, __half> && W > 1) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) reinterpret_cast<__half2*>(a.s)[i] = __hsub2(reinterpret_cast<__half2*>(a.s)[i], reinterpret_cast<const __half2*>(b.s)[i]);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) a.set(i, a.get(i) - b.get(i));
    }
}
template <typename T, int W> __device__ __forceinline__ bool frag_any_above(const Frag<T, W>& a, float thr) {
    if constexpr (std::is_same_v<T, __half> && W > 1) {      // thr is a half already
        const __half2 t = __float2half2_rn(thr);
        unsigned any = 0;
#pragma unroll
        for (int i = 0; i < W / 2; ++i) any |= __hgt2_mask(__habs2(reinterpret_cast<const __half2*>(a.s)[i]), t);
        return any != 0;
    } else {
        bool any = false;
#pragma unroll
        for (int i = 0; i < W; ++i) any |= fabsf(a.get(i)) > thr;
        return any;
    }
}

// What a team reads of a pixel; packs behind the last channel hold zeros.
template <typename T, int W, int P> struct DeltaPixel {
    Frag<T, W> d[P], u[P], o[P];           // the delta, the accumulated input, the accumulated output
    template <bool BLOCK> __device__ __forceinline__ void load(const LnDeltaParams& p, const Team<BLOCK, P>& t, int64_t px, bool on) {
        const int64_t off = px * p.c + t.first * W;
#pragma unroll
        for (int k = 0; k < P; ++k) {
            d[k].fill(0.f); u[k].fill(0.f); o[k].fill(0.f);
            if (on && t.first + k * t.hop() < p.nvec) {
                const int64_t at = off + k * t.hop() * W;
                d[k].load((const T*)p.delta + at);
                u[k].load((const T*)p.prev_in + at);
                o[k].load((const T*)p.prev_out + at);
            }
        }
    }
};
// One pixel by its team; returns whether any channel's change is above the threshold (the same answer in the whole team).
template <typename T, typename WT, int W, int P, bool BLOCK>
__device__ __forceinline__ bool ln_delta_pixel(const LnDeltaParams& p, const Team<BLOCK, P>& t, int64_t px, bool on, DeltaPixel<T, W, P>& v, Frag<WT, W> (&w)[P],
                                               Frag<WT, W> (&b)[P], float* red0, float* red1) {
    const int64_t off = px * p.c + t.first * W;
    Frag<T, W> (&d)[P] = v.d;
    Frag<T, W> (&u)[P] = v.u;
    Frag<T, W> (&o)[P] = v.o;
    bool valid[P];
#pragma unroll
    for (int k = 0; k < P; ++k) valid[k] = t.first + k * t.hop() < p.nvec;
    using V = typename Vals<W>::V;
    constexpr int N = Vals<W>::N;
    Vals<W> x[P];
    V s = V::all(0.f), q = V::all(0.f);
#pragma unroll
    for (int k = 0; k < P; ++k) {
        frag_add(u[k], d[k]);
        if (on && valid[k]) u[k].store((T*)p.prev_in + off + k * t.hop() * W);
        x[k].from(u[k]);
#pragma unroll
        for (int i = 0; i < N; ++i) s = add(s, x[k].v[i]);
    }
    const float m = t.sum(s.sum(), red0) * p.inv_c;
#pragma unroll
    for (int k = 0; k < P; ++k) {
        const V neg = V::all(valid[k] ? -m : 0.f);
#pragma unroll
        for (int i = 0; i < N; ++i) { x[k].v[i] = add(x[k].v[i], neg); q = fma(x[k].v[i], x[k].v[i], q); }
    }
    const float r = rsqrtf(t.sum(q.sum(), red1) * p.inv_c + p.eps);
    const V rr = V::all(r);
    bool hit = false;
#pragma unroll
    for (int k = 0; k < P; ++k) {
        Vals<W> ww, bb;
        ww.from(w[k]);
        bb.from(b[k]);
#pragma unroll
        for (int i = 0; i < N; ++i) x[k].v[i] = fma(mul(x[k].v[i], rr), ww.v[i], bb.v[i]);
        x[k].to(d[k]);               // the norm is rounded to the storage type first, then the difference: e = 0 exactly where nothing changed since this
                                   // kernel, or dc_layer_norm_delta_first with the same split of the row, wrote prev_out
        frag_sub(d[k], o[k]);
        hit |= frag_any_above(d[k], p.thr);
    }
    bool keep;
    if constexpr (BLOCK) keep = __syncthreads_or(hit) != 0;
    else keep = group_any(hit && on, t.size, threadIdx.x & 31);
    if (on && keep) {
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (valid[k]) {
                frag_add(o[k], d[k]);
                d[k].store((T*)p.out + off + k * t.hop() * W);
                o[k].store((T*)p.prev_out + off + k * t.hop() * W);
            }
    }
    return keep;
}

// Teams of lanes: a warp reads the mask of `chunk` pixels at once, lists the active ones and hands them to its teams, so that
// sparse maps cost one coalesced mask read and no idle teams. The next chunk's mask is on its way meanwhile.
template <typename T, typename WT, int W, int P>
__global__ void __launch_bounds__(256, P == 1 ? 4 : W > 2 ? 1 : 3) k_ln_delta(LnDeltaParams p) {
    __shared__ uint8_t list[8][32], kept[8][32];
    grid_dep_launch();
    grid_dep_wait();
    const Team<false, P> t(p.g);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, teams = 32 / p.g;
    const int64_t step = (int64_t)gridDim.x * 8 * p.chunk;
    int64_t base = ((int64_t)blockIdx.x * 8 + warp) * p.chunk;
    const bool mine = lane < p.chunk;
    int32_t next = mine && base + lane < p.npix ? p.mask[base + lane] : 0;
    Frag<WT, W> w[P], b[P];
    load_param<WT, W, P>(w, (const WT*)p.w, t.first, t.hop(), p.nvec, 1.f);
    load_param<WT, W, P>(b, (const WT*)p.b, t.first, t.hop(), p.nvec, 0.f);
    for (; base < p.npix; base += step) {
        const bool act = next != 0;
        next = mine && base + step + lane < p.npix ? p.mask[base + step + lane] : 0;
        const unsigned m = __ballot_sync(DC_FULL, act);
        if (act) list[warp][__popc(m & ((1u << lane) - 1u))] = (uint8_t)lane;
        kept[warp][lane] = 0;
        __syncwarp();
        const int n = __popc(m);
        // the next pixel's reads are on their way while one is normalised, where a lane has the registers for both
        constexpr bool kAhead = P * W * sizeof(T) <= 16;
        DeltaPixel<T, W, P> v, ahead;
        int at = lane / p.g, px = at < n ? list[warp][at] : 0;
        if (n > 0) v.load(p, t, base + px, at < n);
        for (int k = 0; k < n; k += teams) {
            const bool on = at < n;
            const int next_at = at + teams, next_px = next_at < n ? list[warp][next_at] : 0;
            if (kAhead && k + teams < n) ahead.load(p, t, base + next_px, next_at < n);
            const bool keep = ln_delta_pixel<T, WT, W, P, false>(p, t, base + px, on, v, w, b, nullptr, nullptr);
            if (on && t.rank == 0 && keep) kept[warp][px] = 1;
            at = next_at;
            px = next_px;
            if constexpr (kAhead) v = ahead;
            else if (k + teams < n) v.load(p, t, base + px, at < n);
        }
        __syncwarp();
        if (mine && base + lane < p.npix) p.mask_out[base + lane] = kept[warp][lane];
        __syncwarp();
    }
}

template <typename T, typename WT, int W, int P>
__global__ void __launch_bounds__(kLnCta) k_ln_delta_cta(LnDeltaParams p) {
    __shared__ float red[2][kMaxWarps];
    grid_dep_launch();
    grid_dep_wait();
    const Team<true, P> t(0);
    Frag<WT, W> w[P], b[P];
    load_param<WT, W, P>(w, (const WT*)p.w, t.first, t.hop(), p.nvec, 1.f);
    load_param<WT, W, P>(b, (const WT*)p.b, t.first, t.hop(), p.nvec, 0.f);
    int32_t next = t.row < p.npix ? p.mask[t.row] : 0;
    for (int64_t px = t.row; px < p.npix; px += t.stride) {
        const bool act = next != 0;            // the same word in every thread
        next = px + t.stride < p.npix ? p.mask[px + t.stride] : 0;
        bool keep = false;
        if (act) {
            DeltaPixel<T, W, P> v;
            v.load(p, t, px, true);
            keep = ln_delta_pixel<T, WT, W, P, true>(p, t, px, true, v, w, b, red[0], red[1]);
        }
        __syncthreads();                       // mask_out may be mask: everybody has read it
        if (t.rank == 0) p.mask_out[px] = keep ? 1 : 0;
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// How a row of c elements is split: width of an access, packs per thread, threads of the team.
struct LnShape {
    int w, p, g, threads;      // g > 0: lanes of a warp; g == 0: a CTA of `threads`; p == 0: the long loop
};

// warp_packs: most packs per lane of a row that a group of lanes takes (more registers per lane than a CTA's threads need, but
// no barriers). cta_packs: most 16-byte packs per thread of a CTA.
// narrow_packs: as warp_packs, for narrow accesses, where the rows fill every SM's threads.
// access: bytes that the arrays' addresses allow, 16, 4 or less.
static LnShape ln_shape(int c, int64_t rows, int elem_bytes, int access, int warp_packs, int cta_packs, int narrow_packs = 4) {
    LnShape s{};
    const int vec = 16 / elem_bytes;
    // 16-byte packs; two halves where a row's width or place allows no more (half the instructions of single ones); elements
    s.w = access >= 16 && c % vec == 0 ? vec : elem_bytes == 2 && access >= 4 && c % 2 == 0 ? 2 : 1;
    const int n = c / s.w;
    // narrow accesses: at least four per thread, so that a thread has several reads in flight
    const bool wide = s.w == vec;
    if (n <= 32 * (wide ? warp_packs : rows * 32 >= (int64_t)sm_count() * 1024 ? narrow_packs : 4)) {
        s.g = lanes_per_pixel(n);
        // Rows enough for every SM's threads all the same: fewer lanes with more packs each shuffle less per element (96 channels
        // in fp16, 200000 rows: 16 lanes of one pack 25 us, 4 lanes of three 17.8 us).
        while (wide && s.g > 1 && divup(n, s.g / 2) <= warp_packs && rows * (s.g / 2) >= (int64_t)sm_count() * 1024) s.g /= 2;
        // Narrow accesses: as few lanes as four of them each allow, for the reads in flight (delta form, 19 channels in fp32, 64 maps of
        // 130 x 200: 32 lanes of one 125 us, 8 lanes of four 79 us); the forward pass of many rows takes up to eight (332222 x 101 in
        // bf16 74 -> 56 us, 166111 x 202 42 -> 35; sixteen are no faster, and eight are too many beside the backward's sums).
        while (!wide && s.g > 1 && (divup(n, s.g / 2) <= 4 || (divup(n, s.g / 2) <= narrow_packs && rows * (s.g / 2) >= (int64_t)sm_count() * 1024))) s.g /= 2;
        const int need = divup(n, s.g);
        s.p = wide ? need : need <= 4 ? 4 : 8;
        s.threads = 256;
        return s;
    }
    s.p = wide ? (n <= 256 ? 1 : n <= 2 * kLnCta ? 2 : 4) : n <= 512 ? 4 : s.w == 2 || n <= 4096 ? 8 : 16;
    const int threads = divup(divup(n, s.p), 32) * 32;
    if (threads <= kLnCta && (!wide || s.p <= cta_packs)) { s.threads = threads; return s; }
    s.p = 0; s.threads = kLongThreads;
    return s;
}

// CTAs of a kernel that an SM holds; the grid is sized by it, so that every CTA's rows, and its one read of the parameters, start at once.
// The first query of a kernel and CTA size also raises the kernel's limit of dynamic shared memory, whatever this launch needs of it:
// without that a launch gets 48 KB together with the kernel's static memory, and the rings of some widths are 48 KB by themselves.
template <auto KERNEL>
static int resident_ctas(int threads, size_t smem) {
    static int known[64][33] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    int& n = known[dev][threads / 32];
    if (n == 0) {
        int v = 0;
        if ((smem > 0 && cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, kLongSmem) != cudaSuccess) ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&v, KERNEL, threads, smem) != cudaSuccess || v < 1) {
            (void)cudaGetLastError();
            return 1;          // not remembered: the launch tells what is wrong, the next call asks again
        }
        n = v;
    }
    return n;
}

static int64_t ln_ctas(const LnShape& s, int64_t rows, int per_sm) {
    const int64_t want = s.g > 0 ? divup64(rows, s.threads / s.g) : rows;
    const int64_t cap = (int64_t)sm_count() * per_sm;
    return want < cap ? (want < 1 ? 1 : want) : cap;
}

// DC_LN_RUN for the instantiation that a shape names, of those that ln_shape can give.
#define DC_LN_CASE(N, KERNEL, T, WT, W, BLOCK) case N: DC_LN_RUN((KERNEL<T, WT, W, N DC_LN_TAIL(BLOCK)>)); break;
#define DC_LN_PACKS2(KERNEL, T, WT, W, BLOCK) switch (s.p) { DC_LN_CASE(1, KERNEL, T, WT, W, BLOCK) DC_LN_CASE(2, KERNEL, T, WT, W, BLOCK) default: break; }
#define DC_LN_PACKS4(KERNEL, T, WT, W, BLOCK) \
    switch (s.p) { DC_LN_CASE(1, KERNEL, T, WT, W, BLOCK) DC_LN_CASE(2, KERNEL, T, WT, W, BLOCK) DC_LN_CASE(4, KERNEL, T, WT, W, BLOCK) default: break; }
#define DC_LN_PACKS1234(KERNEL, T, WT, W, BLOCK)                                                               \
    switch (s.p) {                                                                                             \
        DC_LN_CASE(1, KERNEL, T, WT, W, BLOCK) DC_LN_CASE(2, KERNEL, T, WT, W, BLOCK)                          \
        DC_LN_CASE(3, KERNEL, T, WT, W, BLOCK) DC_LN_CASE(4, KERNEL, T, WT, W, BLOCK) default: break;          \
    }
// Narrow accesses: single elements (W 1) or two halves (W 2).
#define DC_LN_NARROW4(KERNEL, T, WT, W) switch (s.p) { DC_LN_CASE(4, KERNEL, T, WT, W, false) default: break; }
#define DC_LN_NARROW48(KERNEL, T, WT, W) \
    switch (s.p) { DC_LN_CASE(4, KERNEL, T, WT, W, false) DC_LN_CASE(8, KERNEL, T, WT, W, false) default: break; }
#define DC_LN_SINGLE_CTA(KERNEL, T, WT) \
    switch (s.p) { DC_LN_CASE(4, KERNEL, T, WT, 1, true) DC_LN_CASE(8, KERNEL, T, WT, 1, true) DC_LN_CASE(16, KERNEL, T, WT, 1, true) default: break; }
#define DC_LN_PAIR_CTA(KERNEL, T, WT) switch (s.p) { DC_LN_CASE(4, KERNEL, T, WT, 2, true) DC_LN_CASE(8, KERNEL, T, WT, 2, true) default: break; }
// The kernel of teams of lanes and the one of a CTA per row, for every access.
#define DC_LN_ALL(WARP_KERNEL, WARP_PACKS, NARROW, CTA_KERNEL, CTA_PACKS, T, WT)                                                  \
    if (s.w == V) { if (s.g > 0) { WARP_PACKS(WARP_KERNEL, T, WT, V, false) } else { CTA_PACKS(CTA_KERNEL, T, WT, V, true) } }                   \
    else if (s.w == 1) { if (s.g > 0) { NARROW(WARP_KERNEL, T, WT, 1) } else { DC_LN_SINGLE_CTA(CTA_KERNEL, T, WT) } }              \
    else if constexpr (sizeof(T) == 2) { if (s.g > 0) { NARROW(WARP_KERNEL, T, WT, 2) } else { DC_LN_PAIR_CTA(CTA_KERNEL, T, WT) } }

#define DC_LN_TAIL(BLOCK) , BLOCK
template <auto KERNEL>
static int ln_forward_run(const LnShape& s, LnParams& p, size_t smem, cudaStream_t st) {
    const int64_t ctas = ln_ctas(s, p.rows, resident_ctas<KERNEL>(s.threads, smem));
    return launch_pdl(KERNEL, dim3((unsigned)ctas), dim3(s.threads), smem, st, p);
}
template <typename T, typename WT, int W>
static int ln_forward_long(LnParams& p, cudaStream_t st) {
    const size_t smem = (size_t)p.c * sizeof(T);
    const bool held = smem <= kLongSmem;
    // an SM's 227 KB, of which every CTA takes 1 KB and the sums of its warps besides
    const int fit = held ? (int)(227 * 1024 / (smem + 1536)) : kLongCtas;
    const int64_t cap = (int64_t)sm_count() * (fit < kLongCtas ? fit : kLongCtas);
    const dim3 grid((unsigned)(p.rows < cap ? p.rows : cap));
    if (!held) return launch_pdl(k_ln_fwd_long<T, WT, W, false>, grid, dim3(kLongThreads), 0, st, p);
    (void)resident_ctas<k_ln_fwd_long<T, WT, W, true>>(kLongThreads, kLongSmem);      // sets the shared memory limit once per device
    return launch_pdl(k_ln_fwd_long<T, WT, W, true>, grid, dim3(kLongThreads), smem, st, p);
}
template <typename T, typename WT>
static int ln_forward_t(const LnShape& s, LnParams& p, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const size_t smem = s.w == V ? (size_t)s.threads * s.p * (rows_ahead(s.p) + 1) * 16 : 0;
    int rc = DC_ERR_UNSUPPORTED;
#define DC_LN_RUN(K) rc = ln_forward_run<K>(s, p, smem, st)
    if (s.p == 0) {
        if (s.w == V) return ln_forward_long<T, WT, V>(p, st);
        if constexpr (sizeof(T) == 2) if (s.w == 2) return ln_forward_long<T, WT, 2>(p, st);
        return ln_forward_long<T, WT, 1>(p, st);
    }
    DC_LN_ALL(k_ln_fwd, DC_LN_PACKS1234, DC_LN_NARROW48, k_ln_fwd, DC_LN_PACKS4, T, WT)
#undef DC_LN_RUN
    return rc;
}

// How the backward pass is split: slices of the workspace with a CTA's column sums each (long rows: a block of rows), which depend
// on nothing but the sizes and the GPU; long rows: blocks of columns, rows of a block.
struct LnSplit {
    int64_t slices, per;
    int blocks;
};
static LnSplit ln_split(const LnShape& s, int c, int64_t rows) {
    LnSplit t{0, 0, 1};
    if (s.p > 0) {      // what an SM holds at the kernels' register bounds
        const int per_sm = bwd_ctas(s.w, s.p) * row_threads(s.w, s.p) / s.threads;
        t.slices = ln_ctas(s, rows, per_sm < 1 ? 1 : per_sm);
        return t;
    }
    t.blocks = divup(c / s.w, kColThreads * (s.w >= 4 ? 1 : 4 / s.w));
    const int64_t room = (int64_t)sm_count() * kColCtas / t.blocks;      // one wave of CTAs
    t.per = divup64(rows, room < 1 ? 1 : room);
    if (t.per < kColMinRows) t.per = kColMinRows;
    t.slices = divup64(rows, t.per);
    return t;
}
static size_t ln_means_floats(const LnShape& s, int64_t rows) { return s.p == 0 ? (size_t)rows * 2 : 0; }

template <typename T, typename WT, int W>
static int ln_backward_long(LnBwdParams& p, const LnSplit& t, cudaStream_t st) {
    if (p.dx != nullptr) {
        const int64_t cap = (int64_t)sm_count() * kLongCtas;
        const int rc = launch_pdl(k_ln_bwd_means<T, WT, W>, dim3((unsigned)(p.rows < cap ? p.rows : cap)), dim3(kLongThreads), 0, st, p);
        if (rc != DC_OK) return rc;
    }
    return launch_pdl(k_ln_bwd_cols<T, WT, W>, dim3((unsigned)t.blocks, (unsigned)t.slices), dim3(kColThreads), 0, st, p);
}
template <auto KERNEL>
static int ln_backward_run(const LnShape& s, LnBwdParams& p, int64_t ctas, size_t smem, cudaStream_t st) {
    (void)resident_ctas<KERNEL>(s.threads, smem);          // sets the shared memory limit once per device
    return launch_pdl(KERNEL, dim3((unsigned)ctas), dim3(s.threads), smem, st, p);
}
template <typename T, typename WT>
static int ln_backward_t(const LnShape& s, LnBwdParams& p, const LnSplit& t, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    size_t smem = s.w == V ? (size_t)s.threads * s.p * 2 * (rows_ahead(2 * s.p) + 1) * 16 : 0;
    if (s.g > 0 && smem < (size_t)8 * p.c) smem = (size_t)8 * p.c;
    int rc = DC_ERR_UNSUPPORTED;
#define DC_LN_RUN(K) rc = ln_backward_run<K>(s, p, t.slices, smem, st)
    if (s.p == 0) {
        if (s.w == V) return ln_backward_long<T, WT, V>(p, t, st);
        if constexpr (sizeof(T) == 2) if (s.w == 2) return ln_backward_long<T, WT, 2>(p, t, st);
        return ln_backward_long<T, WT, 1>(p, t, st);
    }
    if constexpr (sizeof(T) == 4) { DC_LN_ALL(k_ln_bwd, DC_LN_PACKS2, DC_LN_NARROW4, k_ln_bwd, DC_LN_PACKS4, T, WT) }
    else { DC_LN_ALL(k_ln_bwd, DC_LN_PACKS2, DC_LN_NARROW4, k_ln_bwd, DC_LN_PACKS2, T, WT) }
#undef DC_LN_RUN
    return rc;
}
#undef DC_LN_TAIL

#define DC_LN_TAIL(BLOCK)
template <auto KERNEL>
static int ln_delta_run(const LnShape& s, LnDeltaParams& p, cudaStream_t st) {
    const int64_t resident = (int64_t)sm_count() * resident_ctas<KERNEL>(s.threads, 0);
    // teams of lanes: pixels that a warp takes at once, at most 32 and so many that every resident warp has as many: with powers
    // of two alone some warps had twice the others' (all active, fp16, 64 x 30 x 40, 320 channels: 98 -> 66 us)
    const int64_t warps = resident * 8, rounds = divup64(p.npix, warps * 32);
    p.chunk = (int)divup64(p.npix, warps * rounds);
    if (p.chunk < 4) p.chunk = 4;
    const int64_t want = s.g > 0 ? divup64(p.npix, p.chunk * 8) : p.npix;
    return launch_pdl(KERNEL, dim3((unsigned)(want < resident ? want : resident)), dim3(s.threads), 0, st, p);
}
template <typename T, typename WT>
static int ln_delta_t(const LnShape& s, LnDeltaParams& p, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    int rc = DC_ERR_UNSUPPORTED;
#define DC_LN_RUN(K) rc = ln_delta_run<K>(s, p, st)
    DC_LN_ALL(k_ln_delta, DC_LN_PACKS1234, DC_LN_NARROW4, k_ln_delta_cta, DC_LN_PACKS4, T, WT)
#undef DC_LN_RUN
    return rc;
}
#undef DC_LN_TAIL

#define DC_LN_TYPES(FN, ...)                                                                                  \
    switch (dtype) {                                                                                          \
        case DC_F32: return weight_dtype == DC_F32 ? FN<float, float>(__VA_ARGS__) : DC_ERR_DTYPE;            \
        case DC_F16: return weight_dtype == DC_F32 ? FN<__half, float>(__VA_ARGS__)                           \
                            : weight_dtype == DC_F16 ? FN<__half, __half>(__VA_ARGS__) : DC_ERR_DTYPE;        \
        case DC_BF16: return weight_dtype == DC_F32 ? FN<__nv_bfloat16, float>(__VA_ARGS__)                   \
                             : weight_dtype == DC_BF16 ? FN<__nv_bfloat16, __nv_bfloat16>(__VA_ARGS__) : DC_ERR_DTYPE; \
        default: return DC_ERR_DTYPE;                                                                         \
    }

static bool ln_dtypes_ok(int dtype, int weight_dtype) {
    return dtype >= DC_F32 && dtype <= DC_BF16 && (weight_dtype == dtype || weight_dtype == DC_F32);
}
static int ln_elem(int dtype) { return dtype == DC_F32 ? 4 : 2; }

// Bytes that an access of the arrays may take: 16, 4, or an element's.
static int ln_access(std::initializer_list<const void*> arrays, const void* weight, const void* bias) {
    uintptr_t a = 0;
    for (const void* p : arrays) a |= reinterpret_cast<uintptr_t>(p);
    return !aligned16(weight) || !aligned16(bias) ? 1 : (a & 15u) == 0 ? 16 : (a & 3u) == 0 ? 4 : 1;
}
// Four packs of eight halves are 64 column sums per thread, which its 128 registers do not hold beside the row: the long kernels'
// two reads are faster (3276 x 10240 in bf16: 87 -> 68 us).
static int bwd_cta_packs(int elem_bytes) { return elem_bytes == 2 ? 2 : 4; }
constexpr int kLnMaxC = 1 << 30;          // a row's places are 32-bit
constexpr int kFwdWarpPacks = 4, kBwdWarpPacks = 2, kDeltaWarpPacks = 4;
static LnShape ln_delta_shape(int c, int dtype, int access) { return ln_shape(c, 0, ln_elem(dtype), access, kDeltaWarpPacks, 4); }

}  // namespace dc

using namespace dc;

extern "C" {

int dc_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, int64_t rows, int32_t c,
                  int32_t dtype, int32_t weight_dtype, float eps, void* stream) {
    if (x == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr)) return DC_ERR_NULL_POINTER;
    if (rows < 0 || c <= 0 || c > kLnMaxC) return DC_ERR_SHAPE;
    if (!ln_dtypes_ok(dtype, weight_dtype)) return DC_ERR_DTYPE;
    if (rows == 0) return DC_OK;
    const LnShape s = ln_shape(c, rows, ln_elem(dtype), ln_access({x, y}, weight, bias), kFwdWarpPacks, 4, 8);
    LnParams p{x, weight, bias, y, mean, rstd, rows, c, c / s.w, s.g, eps, 1.f / (float)c};
    DC_LN_TYPES(ln_forward_t, s, p, (cudaStream_t)stream)
}

size_t dc_layer_norm_backward_workspace_bytes(int64_t rows, int32_t c, int32_t dtype) {
    if (rows <= 0 || c <= 0 || c > kLnMaxC || dtype < DC_F32 || dtype > DC_BF16) return 0;
    // the split may differ with the pointers' alignment: room for any
    size_t most = 0;
    for (int access : {16, 4, 1}) {
        const LnShape s = ln_shape(c, rows, ln_elem(dtype), access, kBwdWarpPacks, bwd_cta_packs(ln_elem(dtype)));
        const size_t n = ln_means_floats(s, rows) + (size_t)ln_split(s, c, rows).slices * 2 * c;
        if (n > most) most = n;
    }
    return most * sizeof(float);
}

int dc_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd, void* dx,
                           void* dweight, void* dbias, int64_t rows, int32_t c, int32_t dtype, int32_t weight_dtype, void* workspace,
                           size_t workspace_bytes, void* stream) {
    if (rows < 0 || c <= 0 || c > kLnMaxC) return DC_ERR_SHAPE;
    if (!ln_dtypes_ok(dtype, weight_dtype)) return DC_ERR_DTYPE;
    const bool sums = dweight != nullptr || dbias != nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) return sums ? col_reduce(nullptr, 0, c, 0, dweight, dbias, weight_dtype, st) : (int)DC_OK;
    if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr) return DC_ERR_NULL_POINTER;
    if (dx == nullptr && !sums) return DC_OK;
    const LnShape s = ln_shape(c, rows, ln_elem(dtype), ln_access({dy, x, dx}, weight, nullptr), kBwdWarpPacks, bwd_cta_packs(ln_elem(dtype)));
    const LnSplit t = ln_split(s, c, rows);
    const size_t means = ln_means_floats(s, rows);
    if (sums || means > 0) {
        if (workspace == nullptr) return DC_ERR_NULL_POINTER;
        if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return DC_ERR_ALIGNMENT;
        if (workspace_bytes < (means + (sums ? (size_t)t.slices * 2 * c : 0)) * sizeof(float)) return DC_ERR_WORKSPACE;
    }
    // the column sums first: their packs want the workspace's alignment
    float* partial = sums ? (float*)workspace : nullptr;
    LnBwdParams p{dy, x, weight, mean, rstd, dx, partial, (float*)workspace + (sums ? t.slices * 2 * c : 0), rows, t.per, c, c / s.w, s.g, 1.f / (float)c};
    const int rc = [&]() -> int { DC_LN_TYPES(ln_backward_t, s, p, t, st) }();
    if (rc != DC_OK || !sums) return rc;
    return col_reduce(partial, (int)t.slices, c, 2 * (int64_t)c, dweight, dbias, weight_dtype, st);
}

// The row is split as below: a pixel that does not change afterwards has the same norm bit for bit. dc_layer_norm's own split may be
// another, since it looks at the number of rows too.
int dc_layer_norm_delta_first(const void* x, const void* weight, const void* bias, void* prev_out, int64_t npix, int32_t c, int32_t dtype,
                              int32_t weight_dtype, float eps, void* stream) {
    if (x == nullptr || prev_out == nullptr) return DC_ERR_NULL_POINTER;
    if (npix < 0 || c <= 0 || c > kLnMaxC) return DC_ERR_SHAPE;
    if (dtype == DC_BF16 || !ln_dtypes_ok(dtype, weight_dtype)) return DC_ERR_DTYPE;
    if (npix == 0) return DC_OK;
    const LnShape s = ln_delta_shape(c, dtype, ln_access({x, prev_out}, weight, bias));
    if (s.p == 0) return DC_ERR_UNSUPPORTED;
    LnParams p{x, weight, bias, prev_out, nullptr, nullptr, npix, c, c / s.w, s.g, eps, 1.f / (float)c};
    DC_LN_TYPES(ln_forward_t, s, p, (cudaStream_t)stream)
}

int dc_layer_norm_delta(const void* delta, const int32_t* mask, void* prev_in, void* prev_out, const void* weight, const void* bias,
                        void* out, int32_t* mask_out, int64_t npix, int32_t c, int32_t dtype, int32_t weight_dtype, float threshold,
                        float eps, void* stream) {
    if (delta == nullptr || mask == nullptr || prev_in == nullptr || prev_out == nullptr || out == nullptr || mask_out == nullptr)
        return DC_ERR_NULL_POINTER;
    if (npix < 0 || c <= 0 || c > kLnMaxC) return DC_ERR_SHAPE;
    if (dtype == DC_BF16 || !ln_dtypes_ok(dtype, weight_dtype)) return DC_ERR_DTYPE;      // the caches are those of the delta path
    if (npix == 0) return DC_OK;
    const LnShape s = ln_delta_shape(c, dtype, ln_access({delta, prev_in, prev_out, out}, weight, bias));
    if (s.p == 0) return DC_ERR_UNSUPPORTED;      // more channels than the registers of a CTA hold
    const float thr = dtype == DC_F16 ? host_round_threshold<__half>(threshold) : threshold;
    LnDeltaParams p{delta, weight, bias, mask, prev_in, prev_out, out, mask_out, npix, c, c / s.w, s.g, thr, eps, 1.f / (float)c, 32};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DC_F32) return ln_delta_t<float, float>(s, p, st);
    return weight_dtype == DC_F32 ? ln_delta_t<__half, float>(s, p, st) : ln_delta_t<__half, __half>(s, p, st);
}

}  // extern "C"
