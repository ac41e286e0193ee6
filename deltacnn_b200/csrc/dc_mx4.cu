// MXFP4 quantisation (blocks along the rows, along the columns, or both from one read) and dequantisation.
//
// Bound: memory. x is read once; a value leaves as half a byte plus 1/32 byte of scale per image.
//
// Rows only (k_mx4_rows): a lane owns eight neighbouring values (one or two 16-byte reads), four lanes a block: the block's
// largest magnitude takes two shuffles, the codes of a lane are one 4-byte store, the scales of four blocks one more.
//
// Both images (k_mx4_tile): a CTA takes 128 x 128 values at a time, which is exactly one 512-byte scale tile of either image,
// and has the next tile on its way into shared memory meanwhile. The rows are encoded as above, the columns two neighbouring
// ones of a 32-row block per thread. Rows 32 apart would meet in the same banks, so every 32 rows are skewed by 16 values:
// a warp reads 8 column pairs x 4 blocks without a conflict and writes 64 contiguous bytes per column. The column sums (the
// bias gradient of a linear layer, whose dy this kernel reads anyway) fall out of the columns' pass.
#include "dc_mx4.cuh"

namespace dc {

int col_reduce(const float* partial, int n, int c, int64_t pitch, void* o0, void* o1, int dtype, cudaStream_t st);   // dc_norm.cu

constexpr int kMxChunk = 256;          // values of a row that a warp takes at once (eight blocks)
constexpr int kMxAhead = 4;            // chunks of a row whose reads a warp has in flight

// A warp's way through rows x segments (a segment: kMxAhead chunks) with the grid's stride: one division at the start, the
// stride's quotient and remainder from the host.
struct MxWalk {
    int segments, step_seg;
    int64_t rows, step_row;
};
static MxWalk mx_walk(int64_t rows, int segments, int64_t warps) { return MxWalk{segments, (int)(warps % segments), rows, warps / segments}; }
struct MxPlace {
    int64_t row;
    int seg;
    __device__ __forceinline__ MxPlace(const MxWalk& w) {
        const int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
        row = it / w.segments;
        seg = (int)(it - row * w.segments);
    }
    __device__ __forceinline__ void next(const MxWalk& w) {
        row += w.step_row;
        seg += w.step_seg;
        if (seg >= w.segments) { seg -= w.segments; ++row; }
    }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_mx4_rows(const T* __restrict__ x, uint8_t* __restrict__ data, uint8_t* __restrict__ scales, int cols, MxWalk w) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31;
    const int nb = (int)mx4_blocks(cols), tiles = (int)mx4_scale_tiles(cols);
    for (MxPlace at(w); at.row < w.rows; at.next(w)) {
        const int c0 = at.seg * (kMxChunk * kMxAhead) + lane * 8;
        const T* row = x + at.row * cols;
        uint8_t* drow = data + at.row * nb * 16;
        uint8_t* srow = scales + mx4_scale_word(at.row, 0, tiles);
        Eight<T> v[kMxAhead];
#pragma unroll
        for (int a = 0; a < kMxAhead; ++a) v[a].template load<VEC>(row, c0 + a * kMxChunk, cols);
#pragma unroll
        for (int a = 0; a < kMxAhead; ++a) {
            const int col = c0 + a * kMxChunk, b = col >> 5;
            uint32_t s;
            const uint32_t code = mx4_encode_lane<T>(v[a], s);
            if (b < nb) *reinterpret_cast<uint32_t*>(drow + (col >> 1)) = code;
            // the scale bytes of four blocks as one word, written by the first lane of every sixteen
            const uint32_t word = mx4_scale_quad(s, lane);
            if ((lane & 15) == 0 && (b >> 2) < tiles) *reinterpret_cast<uint32_t*>(srow + (int64_t)(b >> 2) * 512) = word;
        }
    }
}

constexpr int kTile = 128;             // rows and columns of a tile
template <typename T> __host__ __device__ constexpr int tile_bytes() { return (kTile * kTile + 3 * 16) * (int)sizeof(T); }
template <typename T> __device__ __forceinline__ int tile_at(int r, int c) { return (r * kTile + (r >> 5) * 16 + c) * (int)sizeof(T); }

struct MxTileParams {
    const void* x;
    uint8_t *data, *scales, *data_t, *scales_t;      // either pair may be NULL
    float* colsum;                                   // [ceil(rows / 128)][cols], or NULL
    int64_t rows, cols;
    int tiles_x, tiles_y;
};

// One tile into shared memory, zeros outside the matrix. VEC: asynchronous copies (the caller commits and waits).
template <typename T, bool VEC>
__device__ __forceinline__ void mx4_fetch(const MxTileParams& p, uint8_t* tile, int64_t r0, int64_t c0) {
    constexpr int N = VecTraits<T>::kVec, kPacks = kTile / N;
#pragma unroll 4
    for (int i = threadIdx.x; i < kTile * kPacks; i += 256) {
        const int r = i / kPacks, c = (i % kPacks) * N;
        const T* src = (const T*)p.x + (r0 + r) * p.cols + c0 + c;
        uint8_t* dst = tile + tile_at<T>(r, c);
        if constexpr (VEC) {
            const bool in = r0 + r < p.rows && c0 + c < p.cols;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(in ? src : (const T*)p.x),
                         "r"(in ? 16 : 0) : "memory");
        } else {
            Pack<T, N> v;
#pragma unroll
            for (int j = 0; j < N; ++j) v.s[j] = r0 + r < p.rows && c0 + c + j < p.cols ? src[j] : from_f<T>(0.f);
            v.store(reinterpret_cast<T*>(dst));
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_mx4_tile(MxTileParams p) {
    extern __shared__ __align__(16) uint8_t tiles_smem[];
    __shared__ float sums[4][kTile];
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t nb = mx4_blocks(p.cols), tiles = mx4_scale_tiles(p.cols), nbt = mx4_blocks(p.rows), tiles_t = mx4_scale_tiles(p.rows);
    const int count = p.tiles_x * p.tiles_y;
    if constexpr (VEC) {
        mx4_fetch<T, VEC>(p, tiles_smem, (int64_t)(blockIdx.x / p.tiles_x) * kTile, (int64_t)(blockIdx.x % p.tiles_x) * kTile);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    for (int it = blockIdx.x, buf = 0; it < count; it += gridDim.x, buf ^= VEC ? 1 : 0) {
        const int ty = it / p.tiles_x, tx = it - ty * p.tiles_x;
        const int64_t r0 = (int64_t)ty * kTile, c0 = (int64_t)tx * kTile;
        uint8_t* tile = tiles_smem + buf * tile_bytes<T>();
        if constexpr (VEC) {
            const int nt = it + gridDim.x;
            if (nt < count) mx4_fetch<T, VEC>(p, tiles_smem + (buf ^ 1) * tile_bytes<T>(), (int64_t)(nt / p.tiles_x) * kTile, (int64_t)(nt % p.tiles_x) * kTile);
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 1;" ::: "memory");
        } else {
            mx4_fetch<T, VEC>(p, tile, r0, c0);
        }
        __syncthreads();
        // the rows: sixteen lanes a row (eight values each), so a warp takes two rows at a time
        if (p.data != nullptr) {
            const int lc = (lane & 15) * 8;
#pragma unroll 4
            for (int q = 0; q < kTile / 16; ++q) {
                const int tr = q * 16 + warp * 2 + (lane >> 4);
                const int64_t r = r0 + tr;
                Eight<T> v;
#pragma unroll
                for (int k = 0; k < Eight<T>::kWords / 4; ++k) reinterpret_cast<uint4*>(v.w)[k] = reinterpret_cast<const uint4*>(tile + tile_at<T>(tr, lc))[k];
                uint32_t s;
                const uint32_t code = mx4_encode_lane<T>(v, s);
                if (r < p.rows && (c0 + lc) >> 5 < nb) *reinterpret_cast<uint32_t*>(p.data + r * nb * 16 + ((c0 + lc) >> 1)) = code;
                const uint32_t word = mx4_scale_quad(s, lane);
                if ((lane & 15) == 0 && r < p.rows) *reinterpret_cast<uint32_t*>(p.scales + mx4_scale_word(r, tx, tiles)) = word;
            }
        }
        // the columns: a thread takes two columns of a 32-row block; a warp 8 column pairs x the 4 blocks
        const int pair = warp * 8 + (lane & 7), blk = lane >> 3;
        const uint8_t* col = tile + tile_at<T>(blk * 32, pair * 2);
        uint32_t m[2] = {0u, 0u};
        float sum[2] = {0.f, 0.f};
        uint32_t code[2][4], s[2];
        auto values = [&](int i) {           // row i of the block: both columns
            if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float2*>(col + i * kTile * 4);
            else return word_values<T>(*reinterpret_cast<const uint32_t*>(col + i * kTile * 2));
        };
        if constexpr (sizeof(T) == 4) {
#pragma unroll 8
            for (int i = 0; i < 32; ++i) {
                const float2 f = values(i);
                m[0] = amax_word<float>(m[0], __float_as_uint(f.x));
                m[1] = amax_word<float>(m[1], __float_as_uint(f.y));
            }
        } else {
            uint32_t both = 0u;
#pragma unroll
            for (int i = 0; i < 32; ++i) both = amax_word<T>(both, *reinterpret_cast<const uint32_t*>(col + i * kTile * 2));
            const float2 f = word_values<T>(both);
            m[0] = __float_as_uint(f.x);
            m[1] = __float_as_uint(f.y);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) s[k] = mx4_scale_byte(m[k]);
        const float f0 = mx4_factor(s[0]), f1 = mx4_factor(s[1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float u[2][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float2 f = values(j * 8 + i);
                if (p.colsum != nullptr) { sum[0] += f.x; sum[1] += f.y; }
                mul2(f.x, f.y, f0, f1);
                u[0][i] = f.x;
                u[1][i] = f.y;
            }
            code[0][j] = s[0] == 255u ? 0u : mx4_encode8(u[0]);
            code[1][j] = s[1] == 255u ? 0u : mx4_encode8(u[1]);
        }
        if (p.data_t != nullptr) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int64_t c = c0 + pair * 2 + k, b = (int64_t)ty * 4 + blk;
                if (c < p.cols) {
                    if (b < nbt) *reinterpret_cast<uint4*>(p.data_t + (c * nbt + b) * 16) = make_uint4(code[k][0], code[k][1], code[k][2], code[k][3]);
                    p.scales_t[mx4_scale_word(c, ty, tiles_t) + blk] = (uint8_t)s[k];
                }
            }
        }
        if (p.colsum != nullptr) {
            sums[blk][pair * 2] = sum[0];
            sums[blk][pair * 2 + 1] = sum[1];
            __syncthreads();
            if (threadIdx.x < kTile && c0 + threadIdx.x < p.cols)
                p.colsum[ty * p.cols + c0 + threadIdx.x] =
                    (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
        }
        __syncthreads();          // the tile may be overwritten
    }
}

// The way of k_mx4_rows back: a warp takes four chunks of 256 values of a row, a lane eight codes of each.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                        int cols, MxWalk w) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31;
    const int nb = (int)mx4_blocks(cols), tiles = (int)mx4_scale_tiles(cols);
    for (MxPlace at(w); at.row < w.rows; at.next(w)) {
        const int c0 = at.seg * (kMxChunk * kMxAhead) + lane * 8;
        const uint8_t* row = data + at.row * nb * 16;
        const uint8_t* srow = scales + mx4_scale_word(at.row, 0, tiles);
        T* orow = out + at.row * cols;
        uint32_t code[kMxAhead], s[kMxAhead];
#pragma unroll
        for (int a = 0; a < kMxAhead; ++a) {
            const int col = c0 + a * kMxChunk, b = col >> 5;
            code[a] = b < nb ? *reinterpret_cast<const uint32_t*>(row + (col >> 1)) : 0u;
            s[a] = b < nb ? srow[(int64_t)(b >> 2) * 512 + (b & 3)] : 0u;
        }
#pragma unroll
        for (int a = 0; a < kMxAhead; ++a) {
            const int col = c0 + a * kMxChunk;
            const float f = mx4_scale_value(s[a]);
            T* o = orow + col;
            float v[8];
            mx4_decode8(code[a], v);
#pragma unroll
            for (int i = 0; i < 4; ++i) mul2(v[2 * i], v[2 * i + 1], f, f);
            if constexpr (VEC) {
                constexpr int N = VecTraits<T>::kVec;
#pragma unroll
                for (int k = 0; k < 8 / N; ++k) {
                    Pack<T, N> q;
#pragma unroll
                    for (int i = 0; i < N; ++i) q.set(i, v[k * N + i]);
                    if (col + k * N < cols) q.store(o + k * N);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (col + i < cols) o[i] = from_f<T>(v[i]);
            }
        }
    }
}

template <typename T>
static int quantize_t(const void* x, void* data, void* scales, void* data_t, void* scales_t, float* colsum, int64_t rows, int64_t cols, cudaStream_t st) {
    const bool vec = aligned16(x) && cols % VecTraits<T>::kVec == 0;
    if (data_t == nullptr && colsum == nullptr) {
        const int segments = (int)divup64(mx4_scale_tiles(cols) * 128, kMxChunk * kMxAhead);
        int64_t ctas = divup64(rows * segments, 8);
        const int64_t cap = (int64_t)sm_count() * 5;
        if (ctas > cap) ctas = cap;
        const MxWalk w = mx_walk(rows, segments, ctas * 8);
        if (vec) return launch_pdl(k_mx4_rows<T, true>, dim3((unsigned)ctas), dim3(256), 0, st, (const T*)x, (uint8_t*)data, (uint8_t*)scales, (int)cols, w);
        return launch_pdl(k_mx4_rows<T, false>, dim3((unsigned)ctas), dim3(256), 0, st, (const T*)x, (uint8_t*)data, (uint8_t*)scales, (int)cols, w);
    }
    const int64_t tx = divup64(cols, kTile), ty = divup64(rows, kTile);
    if (tx * ty > 0x3fffffffLL) return DC_ERR_SHAPE;
    MxTileParams p{x, (uint8_t*)data, (uint8_t*)scales, (uint8_t*)data_t, (uint8_t*)scales_t, colsum, rows, cols, (int)tx, (int)ty};
    static PerDeviceOnce once;
    bool* set = once.slot();
    if (set == nullptr) return DC_ERR_LAUNCH;
    if (!*set) {
        if (cudaFuncSetAttribute(k_mx4_tile<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * tile_bytes<T>()) != cudaSuccess ||
            cudaFuncSetAttribute(k_mx4_tile<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, tile_bytes<T>()) != cudaSuccess)
            return check_launch();
        *set = true;
    }
    // VEC: two tiles of shared memory per CTA, the next one on its way while a tile is encoded
    const int64_t cap = (int64_t)sm_count() * (sizeof(T) == 4 ? (vec ? 1 : 3) : (vec ? 3 : 4));
    const dim3 grid((unsigned)(tx * ty < cap ? tx * ty : cap));
    if (vec) return launch_pdl(k_mx4_tile<T, true>, grid, dim3(256), 2 * tile_bytes<T>(), st, p);
    return launch_pdl(k_mx4_tile<T, false>, grid, dim3(256), tile_bytes<T>(), st, p);
}

template <typename T>
static int dequantize_t(const void* data, const void* scales, void* out, int64_t rows, int64_t cols, cudaStream_t st) {
    const int segments = (int)divup64(cols, kMxChunk * kMxAhead);
    int64_t ctas = divup64(rows * segments, 8);
    const int64_t cap = (int64_t)sm_count() * 6;
    if (ctas > cap) ctas = cap;
    const MxWalk w = mx_walk(rows, segments, ctas * 8);
    if (aligned16(out) && cols % VecTraits<T>::kVec == 0)
        return launch_pdl(k_mx4_dequantize<T, true>, dim3((unsigned)ctas), dim3(256), 0, st, (const uint8_t*)data, (const uint8_t*)scales, (T*)out, (int)cols, w);
    return launch_pdl(k_mx4_dequantize<T, false>, dim3((unsigned)ctas), dim3(256), 0, st, (const uint8_t*)data, (const uint8_t*)scales, (T*)out, (int)cols, w);
}

}  // namespace dc

using namespace dc;

extern "C" {

size_t dc_mx4_data_bytes(int64_t rows, int64_t cols) { return rows <= 0 || cols <= 0 ? 0 : (size_t)(rows * mx4_blocks(cols) * 16); }
size_t dc_mx4_scale_bytes(int64_t rows, int64_t cols) { return rows <= 0 || cols <= 0 ? 0 : (size_t)(divup64(rows, 128) * mx4_scale_tiles(cols) * 512); }
size_t dc_mx4_colsum_workspace_bytes(int64_t rows, int64_t cols) { return rows <= 0 || cols <= 0 ? 0 : (size_t)(divup64(rows, kTile) * cols) * sizeof(float); }

int dc_mx4_quantize(const void* x, void* data, void* scales, void* data_t, void* scales_t, void* colsum, int64_t rows, int64_t cols, int32_t dtype,
                    int32_t colsum_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (rows < 0 || cols <= 0 || cols > 0x7ffff000LL) return DC_ERR_SHAPE;
    if (dtype < DC_F32 || dtype > DC_BF16 || (colsum != nullptr && (colsum_dtype < DC_F32 || colsum_dtype > DC_BF16))) return DC_ERR_DTYPE;
    if ((data == nullptr) != (scales == nullptr) || (data_t == nullptr) != (scales_t == nullptr)) return DC_ERR_NULL_POINTER;
    if (data == nullptr && data_t == nullptr && colsum == nullptr) return DC_ERR_NULL_POINTER;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) return colsum != nullptr ? col_reduce(nullptr, 0, (int)cols, 0, colsum, nullptr, colsum_dtype, st) : (int)DC_OK;
    if (x == nullptr) return DC_ERR_NULL_POINTER;
    if (!aligned16(data) || !aligned16(scales) || !aligned16(data_t) || !aligned16(scales_t) || !aligned16(workspace)) return DC_ERR_ALIGNMENT;
    if (colsum != nullptr && workspace == nullptr) return DC_ERR_NULL_POINTER;
    if (colsum != nullptr && workspace_bytes < dc_mx4_colsum_workspace_bytes(rows, cols)) return DC_ERR_WORKSPACE;
    float* part = colsum != nullptr ? (float*)workspace : nullptr;
    int rc;
    switch (dtype) {
        case DC_F32: rc = quantize_t<float>(x, data, scales, data_t, scales_t, part, rows, cols, st); break;
        case DC_F16: rc = quantize_t<__half>(x, data, scales, data_t, scales_t, part, rows, cols, st); break;
        default: rc = quantize_t<__nv_bfloat16>(x, data, scales, data_t, scales_t, part, rows, cols, st); break;
    }
    if (rc != DC_OK || colsum == nullptr) return rc;
    return col_reduce(part, (int)divup64(rows, kTile), (int)cols, cols, colsum, nullptr, colsum_dtype, st);
}

int dc_mx4_dequantize(const void* data, const void* scales, void* out, int64_t rows, int64_t cols, int32_t dtype, void* stream) {
    if (rows < 0 || cols <= 0 || cols > 0x7ffff000LL) return DC_ERR_SHAPE;
    if (dtype < DC_F32 || dtype > DC_BF16) return DC_ERR_DTYPE;
    if (rows == 0) return DC_OK;
    if (data == nullptr || scales == nullptr || out == nullptr) return DC_ERR_NULL_POINTER;
    if (!aligned16(data) || !aligned16(scales)) return DC_ERR_ALIGNMENT;
    cudaStream_t st = (cudaStream_t)stream;
    switch (dtype) {
        case DC_F32: return dequantize_t<float>(data, scales, out, rows, cols, st);
        case DC_F16: return dequantize_t<__half>(data, scales, out, rows, cols, st);
        default: return dequantize_t<__nv_bfloat16>(data, scales, out, rows, cols, st);
    }
}

}  // extern "C"
