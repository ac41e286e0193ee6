// Layer norm over the channel vector of a pixel or token: forward, backward with the column reductions of the weight's
// and bias's gradients, and the delta form with its caches.
//
// Mathematics: mean m = sum x / C, variance v = sum (x - m)^2 / C (two sums over values held in registers: no
// cancellation between large sums), r = 1 / sqrt(v + eps), n = (x - m) r, y = n w + b. Backward, with g = dy w:
// dx = r (g - mean(g) - n mean(g n)), dw = sum_rows dy n, db = sum_rows dy.
//
// Split: a row belongs to a team of threads that keeps it in registers between its one read and its one write: an aligned
// group of lanes while the row has at most 128 packs of 16 bytes (several short rows share a warp, sums are shuffles), a
// whole CTA above that. Teams walk rows with the grid's stride; weight and bias are read once per team and stay in
// registers, and the next row is requested before the sums of the current one are taken, so the memory system always has a
// row per team in flight. Rows whose width or address does not allow 16-byte accesses take the same code with single
// elements; rows beyond the registers of a CTA are read three times by a plain loop.
#include "dc_common.cuh"

namespace dc {

// W consecutive elements in storage precision; 16-byte accesses where the size allows.
template <typename T, int W> struct Frag {
    static constexpr int kBytes = W * (int)sizeof(T);
    alignas(kBytes % 16 == 0 ? 16 : alignof(T)) T s[W];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kBytes % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(s)[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) s[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kBytes % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(s)[i];
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) p[i] = s[i];
        }
    }
    __device__ __forceinline__ float get(int i) const { return to_f<T>(s[i]); }
    __device__ __forceinline__ void set(int i, float x) { s[i] = from_f<T>(x); }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int i = 0; i < W; ++i) set(i, x);
    }
};

constexpr int kLnCta = 512;         // most threads of a CTA that holds a row: 128 registers a thread
constexpr int kMaxWarps = 32;

// A row's team: g lanes of a warp (BLOCK false) or the whole CTA (BLOCK true).
template <bool BLOCK> struct Team {
    int rank, size;            // this thread's place in the team, the team's threads
    int64_t row, stride;       // first row, distance to the next one
    __device__ __forceinline__ Team(int g) {
        if constexpr (BLOCK) {
            rank = threadIdx.x; size = blockDim.x; row = blockIdx.x; stride = gridDim.x;
        } else {
            const int per_cta = blockDim.x / g;
            rank = threadIdx.x & (g - 1); size = g;
            row = (int64_t)blockIdx.x * per_cta + threadIdx.x / g;
            stride = (int64_t)gridDim.x * per_cta;
        }
    }
    // Sum over the team, the same bits in every thread. red: kMaxWarps floats per call site (BLOCK); a site is used again
    // only after another site's barrier.
    __device__ __forceinline__ float sum(float x, float* red) const {
        if constexpr (!BLOCK) return group_sum(x, size);
        x = group_sum(x, 32);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
        __syncthreads();
        const int lane = threadIdx.x & 31;
        return group_sum(lane < (int)(blockDim.x >> 5) ? red[lane] : 0.f, 32);
    }
};

template <typename T, int W, int P>
__device__ __forceinline__ void load_row(Frag<T, W> (&v)[P], const T* p, int rank, int size, int nvec) {
#pragma unroll
    for (int k = 0; k < P; ++k)
        if (rank + k * size < nvec) v[k].load(p + (int64_t)(rank + k * size) * W);
}
template <typename T, int W, int P>
__device__ __forceinline__ void load_param(Frag<T, W> (&v)[P], const T* p, int rank, int size, int nvec, float neutral) {
#pragma unroll
    for (int k = 0; k < P; ++k) {
        if (p == nullptr) v[k].fill(neutral);
        else if (rank + k * size < nvec) v[k].load(p + (rank + k * size) * W);
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
__global__ void __launch_bounds__(BLOCK ? kLnCta : 256) k_ln_fwd(LnParams p) {
    __shared__ float red[2][kMaxWarps];
    grid_dep_launch();
    grid_dep_wait();
    const Team<BLOCK> t(p.g);
    const T* x = (const T*)p.x;
    T* y = (T*)p.y;
    Frag<WT, W> w[P], b[P];
    load_param<WT, W, P>(w, (const WT*)p.w, t.rank, t.size, p.nvec, 1.f);
    load_param<WT, W, P>(b, (const WT*)p.b, t.rank, t.size, p.nvec, 0.f);
    Frag<T, W> nx[P];
    if (t.row < p.rows) load_row<T, W, P>(nx, x + t.row * p.c, t.rank, t.size, p.nvec);
    // lanes of a warp whose own rows have run out still take part in its shuffles
    for (int64_t base = t.row - (BLOCK ? 0 : (threadIdx.x & 31) / p.g); base < p.rows; base += t.stride) {
        const int64_t row = BLOCK ? base : base + (threadIdx.x & 31) / p.g;
        const bool on = row < p.rows;
        Frag<T, W> v[P];
#pragma unroll
        for (int k = 0; k < P; ++k) v[k] = nx[k];
        if (row + t.stride < p.rows) load_row<T, W, P>(nx, x + (row + t.stride) * p.c, t.rank, t.size, p.nvec);
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (t.rank + k * t.size < p.nvec)
#pragma unroll
                for (int i = 0; i < W; ++i) s += v[k].get(i);
        const float m = t.sum(s, red[0]) * p.inv_c;
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (t.rank + k * t.size < p.nvec)
#pragma unroll
                for (int i = 0; i < W; ++i) { const float d = v[k].get(i) - m; q += d * d; }
        const float r = __frsqrt_rn(t.sum(q, red[1]) * p.inv_c + p.eps);
        if (on) {
#pragma unroll
            for (int k = 0; k < P; ++k)
                if (t.rank + k * t.size < p.nvec) {
#pragma unroll
                    for (int i = 0; i < W; ++i) v[k].set(i, (v[k].get(i) - m) * r * w[k].get(i) + b[k].get(i));
                    v[k].store(y + row * p.c + (int64_t)(t.rank + k * t.size) * W);
                }
            if (t.rank == 0 && p.mean != nullptr) { p.mean[row] = m; p.rstd[row] = r; }
        }
    }
}

// Rows beyond the registers of a CTA: three reads (the second and third mostly from L2).
template <typename T, typename WT>
__global__ void __launch_bounds__(1024) k_ln_fwd_long(LnParams p) {
    __shared__ float red[2][kMaxWarps];
    grid_dep_launch();
    grid_dep_wait();
    const Team<true> t(0);
    const WT *w = (const WT*)p.w, *b = (const WT*)p.b;
    for (int64_t row = t.row; row < p.rows; row += t.stride) {
        const T* x = (const T*)p.x + row * p.c;
        T* y = (T*)p.y + row * p.c;
        float s = 0.f;
        for (int i = t.rank; i < p.c; i += t.size) s += to_f<T>(x[i]);
        const float m = t.sum(s, red[0]) * p.inv_c;
        float q = 0.f;
        for (int i = t.rank; i < p.c; i += t.size) { const float d = to_f<T>(x[i]) - m; q += d * d; }
        const float r = __frsqrt_rn(t.sum(q, red[1]) * p.inv_c + p.eps);
        for (int i = t.rank; i < p.c; i += t.size)
            y[i] = from_f<T>((to_f<T>(x[i]) - m) * r * (w != nullptr ? to_f<WT>(w[i]) : 1.f) + (b != nullptr ? to_f<WT>(b[i]) : 0.f));
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
    float* partial;            // [gridDim.x][2][c]: this CTA's sums of dy n and dy; NULL: not wanted
    int64_t rows;
    int c, nvec, g;
    float inv_c;
};

template <typename T, typename WT, int W, int P, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? kLnCta : 256) k_ln_bwd(LnBwdParams p) {
    __shared__ float red[2][2][kMaxWarps];
    extern __shared__ float cols[];            // [2][c]: the CTA's column sums (teams within a CTA only)
    grid_dep_launch();
    grid_dep_wait();
    const Team<BLOCK> t(p.g);
    const T *x = (const T*)p.x, *dy = (const T*)p.dy;
    T* dx = (T*)p.dx;
    Frag<WT, W> w[P];
    load_param<WT, W, P>(w, (const WT*)p.w, t.rank, t.size, p.nvec, 1.f);
    float dw[P][W], db[P][W];
#pragma unroll
    for (int k = 0; k < P; ++k)
#pragma unroll
        for (int i = 0; i < W; ++i) dw[k][i] = db[k][i] = 0.f;
    // four packs a thread leave no registers for the next row; the CTA that holds such a row has 64 KB of it in flight anyway
    constexpr bool kAhead = P * W < 32;
    Frag<T, W> nx[P], nd[P];
    float nm = 0.f, nr = 0.f;
    [[maybe_unused]] int par = 0;
    if (kAhead && t.row < p.rows) {
        load_row<T, W, P>(nx, x + t.row * p.c, t.rank, t.size, p.nvec);
        load_row<T, W, P>(nd, dy + t.row * p.c, t.rank, t.size, p.nvec);
        nm = p.mean[t.row]; nr = p.rstd[t.row];
    }
    for (int64_t base = t.row - (BLOCK ? 0 : (threadIdx.x & 31) / p.g); base < p.rows; base += t.stride) {
        const int64_t row = BLOCK ? base : base + (threadIdx.x & 31) / p.g;
        const bool on = row < p.rows;
        Frag<T, W> v[P], d[P];
        if (!kAhead && on) {
            load_row<T, W, P>(nx, x + row * p.c, t.rank, t.size, p.nvec);
            load_row<T, W, P>(nd, dy + row * p.c, t.rank, t.size, p.nvec);
            nm = p.mean[row]; nr = p.rstd[row];
        }
        const float m = nm, r = nr;
#pragma unroll
        for (int k = 0; k < P; ++k) { v[k] = nx[k]; d[k] = nd[k]; }
        if (kAhead && row + t.stride < p.rows) {
            load_row<T, W, P>(nx, x + (row + t.stride) * p.c, t.rank, t.size, p.nvec);
            load_row<T, W, P>(nd, dy + (row + t.stride) * p.c, t.rank, t.size, p.nvec);
            nm = p.mean[row + t.stride]; nr = p.rstd[row + t.stride];
        }
        float sg = 0.f, sgn = 0.f;
        if (on) {
#pragma unroll
            for (int k = 0; k < P; ++k)
                if (t.rank + k * t.size < p.nvec)
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const float n = (v[k].get(i) - m) * r, e = d[k].get(i), g = e * w[k].get(i);
                        dw[k][i] += e * n;
                        db[k][i] += e;
                        sg += g;
                        sgn += g * n;
                    }
        }
        if (dx != nullptr) {
            float a, c;
            if constexpr (BLOCK) {             // both sums behind one barrier
                const int lane = threadIdx.x & 31;
                par ^= 1;
                sg = group_sum(sg, 32);
                sgn = group_sum(sgn, 32);
                if (lane == 0) { red[par][0][threadIdx.x >> 5] = sg; red[par][1][threadIdx.x >> 5] = sgn; }
                __syncthreads();
                const bool in = lane < (int)(blockDim.x >> 5);
                a = group_sum(in ? red[par][0][lane] : 0.f, 32) * p.inv_c;
                c = group_sum(in ? red[par][1][lane] : 0.f, 32) * p.inv_c;
            } else {
                a = group_sum(sg, t.size) * p.inv_c;
                c = group_sum(sgn, t.size) * p.inv_c;
            }
            if (on) {
#pragma unroll
                for (int k = 0; k < P; ++k)
                    if (t.rank + k * t.size < p.nvec) {
#pragma unroll
                        for (int i = 0; i < W; ++i) {
                            const float n = (v[k].get(i) - m) * r;
                            d[k].set(i, r * (d[k].get(i) * w[k].get(i) - a - n * c));
                        }
                        d[k].store(dx + row * p.c + (int64_t)(t.rank + k * t.size) * W);
                    }
            }
        }
    }
    if (p.partial == nullptr) return;
    float* out = p.partial + (int64_t)blockIdx.x * 2 * p.c;
    if constexpr (BLOCK) {
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (t.rank + k * t.size < p.nvec)
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const int col = (t.rank + k * t.size) * W + i;
                    out[col] = dw[k][i];
                    out[p.c + col] = db[k][i];
                }
    } else {
        // teams of a warp by shuffles, warps of the CTA one after the other: a fixed order
#pragma unroll
        for (int k = 0; k < P; ++k)
#pragma unroll
            for (int i = 0; i < W; ++i)
                for (int o = p.g; o < 32; o <<= 1) {
                    dw[k][i] += __shfl_xor_sync(DC_FULL, dw[k][i], o);
                    db[k][i] += __shfl_xor_sync(DC_FULL, db[k][i], o);
                }
        const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        for (int q = 0; q < warps; ++q) {
            if (warp == q && (threadIdx.x & 31) < p.g) {
#pragma unroll
                for (int k = 0; k < P; ++k)
                    if (t.rank + k * t.size < p.nvec)
#pragma unroll
                        for (int i = 0; i < W; ++i) {
                            const int col = (t.rank + k * t.size) * W + i;
                            cols[col] = (q == 0 ? 0.f : cols[col]) + dw[k][i];
                            cols[p.c + col] = (q == 0 ? 0.f : cols[p.c + col]) + db[k][i];
                        }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 2 * p.c; i += blockDim.x) out[i] = cols[i];
    }
}

// Long rows: the row's two sums in a first loop, dx in a second; the column sums go through the CTA's own slice of the
// workspace, whose columns belong to one thread each.
template <typename T, typename WT>
__global__ void __launch_bounds__(1024) k_ln_bwd_long(LnBwdParams p) {
    __shared__ float red[2][kMaxWarps];
    grid_dep_launch();
    grid_dep_wait();
    const Team<true> t(0);
    const WT* w = (const WT*)p.w;
    float* out = p.partial == nullptr ? nullptr : p.partial + (int64_t)blockIdx.x * 2 * p.c;
    if (out != nullptr)
        for (int i = t.rank; i < p.c; i += t.size) out[i] = out[p.c + i] = 0.f;
    for (int64_t row = t.row; row < p.rows; row += t.stride) {
        const T *x = (const T*)p.x + row * p.c, *dy = (const T*)p.dy + row * p.c;
        const float m = p.mean[row], r = p.rstd[row];
        float sg = 0.f, sgn = 0.f;
        for (int i = t.rank; i < p.c; i += t.size) {
            const float n = (to_f<T>(x[i]) - m) * r, e = to_f<T>(dy[i]), g = e * (w != nullptr ? to_f<WT>(w[i]) : 1.f);
            if (out != nullptr) { out[i] += e * n; out[p.c + i] += e; }
            sg += g;
            sgn += g * n;
        }
        const float a = t.sum(sg, red[0]) * p.inv_c, c = t.sum(sgn, red[1]) * p.inv_c;
        if (p.dx != nullptr) {
            T* dx = (T*)p.dx + row * p.c;
            for (int i = t.rank; i < p.c; i += t.size) {
                const float n = (to_f<T>(x[i]) - m) * r;
                dx[i] = from_f<T>(r * (to_f<T>(dy[i]) * (w != nullptr ? to_f<WT>(w[i]) : 1.f) - a - n * c));
            }
        }
    }
}

// Column sums of the CTAs' partial rows, in a fixed order: 32 columns per CTA, 16 threads share a column's rows.
constexpr int kRedRows = 16;
template <typename OT>
__global__ void __launch_bounds__(32 * kRedRows) k_col_reduce(const float* __restrict__ partial, int n, int c, int64_t pitch, OT* __restrict__ o0,
                                                              OT* __restrict__ o1) {
    __shared__ float s[kRedRows][33];
    grid_dep_launch();
    grid_dep_wait();
    const int col = blockIdx.x * 32 + threadIdx.x;
    OT* o = blockIdx.y == 0 ? o0 : o1;
    if (o == nullptr) return;
    float a = 0.f;
    if (col < c)
        for (int i = threadIdx.y; i < n; i += kRedRows) a += partial[i * pitch + (int64_t)blockIdx.y * c + col];
    s[threadIdx.y][threadIdx.x] = a;
    __syncthreads();
    if (threadIdx.y == 0 && col < c) {
        a = 0.f;
#pragma unroll
        for (int i = 0; i < kRedRows; ++i) a += s[i][threadIdx.x];
        o[col] = from_f<OT>(a);
    }
}

int col_reduce(const float* partial, int n, int c, int64_t pitch, void* o0, void* o1, int dtype, cudaStream_t st) {
    const dim3 grid((unsigned)divup(c, 32), o1 != nullptr ? 2u : 1u), block(32, kRedRows);
    switch (dtype) {
        case DC_F32: return launch_pdl(k_col_reduce<float>, grid, block, 0, st, partial, n, c, pitch, (float*)o0, (float*)o1);
        case DC_F16: return launch_pdl(k_col_reduce<__half>, grid, block, 0, st, partial, n, c, pitch, (__half*)o0, (__half*)o1);
        case DC_BF16: return launch_pdl(k_col_reduce<__nv_bfloat16>, grid, block, 0, st, partial, n, c, pitch, (__nv_bfloat16*)o0, (__nv_bfloat16*)o1);
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
};

// One pixel by its team; returns whether any channel's change is above the threshold (the same answer in the whole team).
template <typename T, typename WT, int W, int P, bool BLOCK>
__device__ __forceinline__ bool ln_delta_pixel(const LnDeltaParams& p, const Team<BLOCK>& t, int64_t px, bool on, Frag<WT, W> (&w)[P], Frag<WT, W> (&b)[P],
                                               float* red0, float* red1) {
    const int64_t off = px * p.c;
    Frag<T, W> u[P], d[P], o[P];
    if (on) {
        load_row<T, W, P>(d, (const T*)p.delta + off, t.rank, t.size, p.nvec);
        load_row<T, W, P>(u, (const T*)p.prev_in + off, t.rank, t.size, p.nvec);
        load_row<T, W, P>(o, (const T*)p.prev_out + off, t.rank, t.size, p.nvec);
    }
    float s = 0.f;
    if (on) {
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (t.rank + k * t.size < p.nvec) {
#pragma unroll
                for (int i = 0; i < W; ++i) { u[k].set(i, u[k].get(i) + d[k].get(i)); s += u[k].get(i); }
                u[k].store((T*)p.prev_in + off + (int64_t)(t.rank + k * t.size) * W);
            }
    }
    const float m = t.sum(s, red0) * p.inv_c;
    float q = 0.f;
    if (on) {
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (t.rank + k * t.size < p.nvec)
#pragma unroll
                for (int i = 0; i < W; ++i) { const float e = u[k].get(i) - m; q += e * e; }
    }
    const float r = __frsqrt_rn(t.sum(q, red1) * p.inv_c + p.eps);
    bool hit = false;
    if (on) {
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (t.rank + k * t.size < p.nvec)
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    // the norm is rounded to the storage type first, then the difference: e = 0 exactly where nothing changed
                    const float y = rnd<T>((u[k].get(i) - m) * r * w[k].get(i) + b[k].get(i));
                    d[k].set(i, y - o[k].get(i));
                    hit |= fabsf(d[k].get(i)) > p.thr;
                }
    }
    bool keep;
    if constexpr (BLOCK) keep = __syncthreads_or(hit) != 0;
    else keep = group_any(hit, t.size, threadIdx.x & 31);
    if (on && keep) {
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (t.rank + k * t.size < p.nvec) {
                const int64_t at = off + (int64_t)(t.rank + k * t.size) * W;
#pragma unroll
                for (int i = 0; i < W; ++i) o[k].set(i, o[k].get(i) + d[k].get(i));
                d[k].store((T*)p.out + at);
                o[k].store((T*)p.prev_out + at);
            }
    }
    return keep;
}

// Teams of lanes: a warp reads the mask of 32 pixels at once, lists the active ones and hands them to its teams, so that
// sparse maps cost one coalesced mask read and no idle teams.
template <typename T, typename WT, int W, int P>
__global__ void __launch_bounds__(256) k_ln_delta(LnDeltaParams p) {
    __shared__ uint8_t list[8][32], kept[8][32];
    grid_dep_launch();
    grid_dep_wait();
    Team<false> t(p.g);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, teams = 32 / p.g;
    Frag<WT, W> w[P], b[P];
    load_param<WT, W, P>(w, (const WT*)p.w, t.rank, t.size, p.nvec, 1.f);
    load_param<WT, W, P>(b, (const WT*)p.b, t.rank, t.size, p.nvec, 0.f);
    const int64_t step = (int64_t)gridDim.x * 8 * 32;
    for (int64_t base = ((int64_t)blockIdx.x * 8 + warp) * 32; base < p.npix; base += step) {
        const bool act = base + lane < p.npix && p.mask[base + lane] != 0;
        const unsigned m = __ballot_sync(DC_FULL, act);
        if (act) list[warp][__popc(m & ((1u << lane) - 1u))] = (uint8_t)lane;
        kept[warp][lane] = 0;
        __syncwarp();
        const int n = __popc(m);
        for (int k = 0; k < n; k += teams) {
            const int at = k + lane / p.g;
            const bool on = at < n;
            const int px = on ? list[warp][at] : 0;
            const bool keep = ln_delta_pixel<T, WT, W, P, false>(p, t, base + px, on, w, b, nullptr, nullptr);
            if (on && t.rank == 0 && keep) kept[warp][px] = 1;
        }
        __syncwarp();
        if (base + lane < p.npix) p.mask_out[base + lane] = kept[warp][lane];
        __syncwarp();
    }
}

template <typename T, typename WT, int W, int P>
__global__ void __launch_bounds__(kLnCta) k_ln_delta_cta(LnDeltaParams p) {
    __shared__ float red[2][kMaxWarps];
    grid_dep_launch();
    grid_dep_wait();
    const Team<true> t(0);
    Frag<WT, W> w[P], b[P];
    load_param<WT, W, P>(w, (const WT*)p.w, t.rank, t.size, p.nvec, 1.f);
    load_param<WT, W, P>(b, (const WT*)p.b, t.rank, t.size, p.nvec, 0.f);
    for (int64_t px = t.row; px < p.npix; px += t.stride) {
        const bool act = p.mask[px] != 0;      // the same word in every thread
        const bool keep = act && ln_delta_pixel<T, WT, W, P, true>(p, t, px, true, w, b, red[0], red[1]);
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

static LnShape ln_shape(int c, int elem_bytes, bool aligned) {
    LnShape s{};
    const int vec = 16 / elem_bytes;
    s.w = aligned && c % vec == 0 ? vec : 1;
    const int n = c / s.w;
    // single elements: eight per thread, so that a thread has as many bytes in flight as a packed one
    const int warp_max = s.w > 1 ? 4 : 8;
    if (n <= 32 * warp_max) {
        s.g = lanes_per_pixel(n);
        const int need = divup(n, s.g);
        s.p = s.w == 1 ? (need <= 2 ? 2 : 8) : need <= 1 ? 1 : need <= 2 ? 2 : 4;
        s.threads = 256;
        return s;
    }
    s.p = s.w == 1 ? 8 : n <= 256 ? 1 : n <= 2 * kLnCta ? 2 : 4;
    const int threads = divup(divup(n, s.p), 32) * 32;
    if (threads <= kLnCta) { s.threads = threads; return s; }
    s.w = 1; s.p = 0; s.threads = 1024;
    return s;
}

static int64_t ln_grid(const LnShape& s, int64_t rows, int per_sm_threads) {
    const int64_t want = s.g > 0 ? divup64(rows, s.threads / s.g) : rows;
    int per_sm = per_sm_threads / s.threads;
    if (per_sm < 1) per_sm = 1;
    const int64_t cap = (int64_t)sm_count() * per_sm;
    return want < cap ? (want < 1 ? 1 : want) : cap;
}

#define DC_LN_P(KERNEL, T, WT, W, BLOCK)                                                  \
    switch (s.p) {                                                                        \
        case 1: DC_LN_RUN((KERNEL<T, WT, W, 1 DC_LN_TAIL(BLOCK)>)); break;                \
        case 2: DC_LN_RUN((KERNEL<T, WT, W, 2 DC_LN_TAIL(BLOCK)>)); break;                \
        case 4: DC_LN_RUN((KERNEL<T, WT, W, 4 DC_LN_TAIL(BLOCK)>)); break;                \
        default: break;                                                                   \
    }
#define DC_LN_P1(KERNEL, T, WT, BLOCK)                                                    \
    switch (s.p) {                                                                        \
        case 2: DC_LN_RUN((KERNEL<T, WT, 1, 2 DC_LN_TAIL(BLOCK)>)); break;                \
        case 8: DC_LN_RUN((KERNEL<T, WT, 1, 8 DC_LN_TAIL(BLOCK)>)); break;                \
        default: break;                                                                   \
    }

#define DC_LN_TAIL(BLOCK) , BLOCK
template <typename T, typename WT>
static int ln_forward_t(const LnShape& s, LnParams& p, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    // 2048 threads a SM is the most it holds; a team prefetches one row, so more resident threads are more rows in flight
    const dim3 grid((unsigned)ln_grid(s, p.rows, 2048)), block(s.threads);
    int rc = DC_ERR_UNSUPPORTED;
#define DC_LN_RUN(K) rc = launch_pdl(K, grid, block, 0, st, p)
    if (s.p == 0) return launch_pdl(k_ln_fwd_long<T, WT>, grid, block, 0, st, p);
    if (s.w > 1) { if (s.g > 0) { DC_LN_P(k_ln_fwd, T, WT, V, false) } else { DC_LN_P(k_ln_fwd, T, WT, V, true) } }
    else { if (s.g > 0) { DC_LN_P1(k_ln_fwd, T, WT, false) } else { DC_LN_P1(k_ln_fwd, T, WT, true) } }
#undef DC_LN_RUN
    return rc;
}

template <typename T, typename WT>
static int ln_backward_t(const LnShape& s, LnBwdParams& p, int64_t ctas, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const dim3 grid((unsigned)ctas), block(s.threads);
    const size_t smem = s.g > 0 ? (size_t)2 * p.c * sizeof(float) : 0;     // at most 2 * 1024 floats
    int rc = DC_ERR_UNSUPPORTED;
#define DC_LN_RUN(K) rc = launch_pdl(K, grid, block, smem, st, p)
    if (s.p == 0) return launch_pdl(k_ln_bwd_long<T, WT>, grid, block, 0, st, p);
    if (s.w > 1) { if (s.g > 0) { DC_LN_P(k_ln_bwd, T, WT, V, false) } else { DC_LN_P(k_ln_bwd, T, WT, V, true) } }
    else { if (s.g > 0) { DC_LN_P1(k_ln_bwd, T, WT, false) } else { DC_LN_P1(k_ln_bwd, T, WT, true) } }
#undef DC_LN_RUN
    return rc;
}
#undef DC_LN_TAIL

#define DC_LN_TAIL(BLOCK)
template <typename T, typename WT>
static int ln_delta_t(const LnShape& s, LnDeltaParams& p, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    int64_t ctas = s.g > 0 ? divup64(p.npix, 256) : p.npix;
    const int64_t cap = (int64_t)sm_count() * (2048 / s.threads > 0 ? 2048 / s.threads : 1);
    if (ctas > cap) ctas = cap;
    const dim3 grid((unsigned)ctas), block(s.threads);
    int rc = DC_ERR_UNSUPPORTED;
#define DC_LN_RUN(K) rc = launch_pdl(K, grid, block, 0, st, p)
    if (s.w > 1) { if (s.g > 0) { DC_LN_P(k_ln_delta, T, WT, V, ) } else { DC_LN_P(k_ln_delta_cta, T, WT, V, ) } }
    else { if (s.g > 0) { DC_LN_P1(k_ln_delta, T, WT, ) } else { DC_LN_P1(k_ln_delta_cta, T, WT, ) } }
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

// CTAs of the backward kernel; each owns a slice of the workspace, so the count depends on nothing but the sizes and the GPU.
static int64_t ln_backward_ctas(const LnShape& s, int64_t rows) { return ln_grid(s, rows, 1024); }

}  // namespace dc

using namespace dc;

extern "C" {

int dc_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, int64_t rows, int32_t c,
                  int32_t dtype, int32_t weight_dtype, float eps, void* stream) {
    if (x == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr)) return DC_ERR_NULL_POINTER;
    if (rows < 0 || c <= 0) return DC_ERR_SHAPE;
    if (!ln_dtypes_ok(dtype, weight_dtype)) return DC_ERR_DTYPE;
    if (rows == 0) return DC_OK;
    const LnShape s = ln_shape(c, ln_elem(dtype), aligned16(x) && aligned16(y) && aligned16(weight) && aligned16(bias));
    LnParams p{x, weight, bias, y, mean, rstd, rows, c, c / s.w, s.g, eps, 1.f / (float)c};
    DC_LN_TYPES(ln_forward_t, s, p, (cudaStream_t)stream)
}

size_t dc_layer_norm_backward_workspace_bytes(int64_t rows, int32_t c, int32_t dtype) {
    if (rows <= 0 || c <= 0 || dtype < DC_F32 || dtype > DC_BF16) return 0;
    // the split may differ with the pointers' alignment: room for either
    const int64_t a = ln_backward_ctas(ln_shape(c, ln_elem(dtype), true), rows), b = ln_backward_ctas(ln_shape(c, ln_elem(dtype), false), rows);
    return (size_t)((a > b ? a : b) * 2 * c) * sizeof(float);
}

int dc_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd, void* dx,
                           void* dweight, void* dbias, int64_t rows, int32_t c, int32_t dtype, int32_t weight_dtype, void* workspace,
                           size_t workspace_bytes, void* stream) {
    if (rows < 0 || c <= 0) return DC_ERR_SHAPE;
    if (!ln_dtypes_ok(dtype, weight_dtype)) return DC_ERR_DTYPE;
    const bool sums = dweight != nullptr || dbias != nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) return sums ? col_reduce(nullptr, 0, c, 0, dweight, dbias, weight_dtype, st) : (int)DC_OK;
    if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr || (sums && workspace == nullptr)) return DC_ERR_NULL_POINTER;
    if (dx == nullptr && !sums) return DC_OK;
    if (sums && (reinterpret_cast<uintptr_t>(workspace) & 3u) != 0) return DC_ERR_ALIGNMENT;
    const LnShape s = ln_shape(c, ln_elem(dtype), aligned16(dy) && aligned16(x) && aligned16(dx) && aligned16(weight));
    const int64_t ctas = ln_backward_ctas(s, rows);
    if (sums && workspace_bytes < (size_t)(ctas * 2 * c) * sizeof(float)) return DC_ERR_WORKSPACE;
    LnBwdParams p{dy, x, weight, mean, rstd, dx, sums ? (float*)workspace : nullptr, rows, c, c / s.w, s.g, 1.f / (float)c};
    const int rc = [&]() -> int { DC_LN_TYPES(ln_backward_t, s, p, ctas, st) }();
    if (rc != DC_OK || !sums) return rc;
    return col_reduce((const float*)workspace, (int)ctas, c, 2 * (int64_t)c, dweight, dbias, weight_dtype, st);
}

int dc_layer_norm_delta(const void* delta, const int32_t* mask, void* prev_in, void* prev_out, const void* weight, const void* bias,
                        void* out, int32_t* mask_out, int64_t npix, int32_t c, int32_t dtype, int32_t weight_dtype, float threshold,
                        float eps, void* stream) {
    if (delta == nullptr || mask == nullptr || prev_in == nullptr || prev_out == nullptr || out == nullptr || mask_out == nullptr)
        return DC_ERR_NULL_POINTER;
    if (npix < 0 || c <= 0) return DC_ERR_SHAPE;
    if (dtype == DC_BF16 || !ln_dtypes_ok(dtype, weight_dtype)) return DC_ERR_DTYPE;      // the caches are those of the delta path
    if (npix == 0) return DC_OK;
    const LnShape s = ln_shape(c, ln_elem(dtype), aligned16(delta) && aligned16(prev_in) && aligned16(prev_out) && aligned16(out) &&
                                                      aligned16(weight) && aligned16(bias));
    if (s.p == 0) return DC_ERR_UNSUPPORTED;      // more channels than the registers of a CTA hold
    const float thr = dtype == DC_F16 ? host_round_threshold<__half>(threshold) : threshold;
    LnDeltaParams p{delta, weight, bias, mask, prev_in, prev_out, out, mask_out, npix, c, c / s.w, s.g, thr, eps, 1.f / (float)c};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DC_F32) return ln_delta_t<float, float>(s, p, st);
    return weight_dtype == DC_F32 ? ln_delta_t<__half, float>(s, p, st) : ln_delta_t<__half, __half>(s, p, st);
}

}  // extern "C"
