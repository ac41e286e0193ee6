// MXFP4 quantisation (blocks along the rows, along the columns, or both from one read) and dequantisation.
//
// Bound: memory. x is read once; a value leaves as half a byte plus 1/32 byte of scale per image.
//
// Rows only (k_mx4_rows): a lane owns eight neighbouring values (one or two 16-byte reads), four lanes a block: the block's
// largest magnitude takes two shuffles, the codes of a lane are one 4-byte store, the scales of four blocks one more.
//
// Both images (k_mx4_tile): a CTA takes 128 x 128 values at a time, which is exactly one 512-byte scale tile of either image,
// and has the next tile on its way into shared memory meanwhile. A lane encodes a whole block of a row (no shuffles, the scale's
// arithmetic once per 32 values), then two neighbouring columns of a 32-row block; a warp writes 64 contiguous bytes per
// column. The column sums (the bias gradient of a linear layer, whose dy this kernel reads anyway) fall out of the columns' pass.
//
// Measured (bf16): rows only, 8192 x 4096, 18 us (85 MB: 13 us at the copy rate); both images of 8192 x 5120 30 us (128 MB: 20 us;
// 50 us with four lanes a block and no tile ahead), issue slots 64 % busy; dequantising 8192 x 5120 18 us (106 MB: 16 us).
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

template <typename T, int BYTES>
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
        for (int a = 0; a < kMxAhead; ++a) v[a].template load<BYTES>(row, c0 + a * kMxChunk, cols);
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
// Where a value of the tile stands: rows in 16-byte pieces, the pieces of a row exchanged so that eight lanes that read the
// same piece of four blocks of two rows, and the eight column pairs x four 32-row blocks of a warp (the rows' skew of 16
// values per 32 rows), meet in no bank.
template <typename T> __host__ __device__ constexpr int tile_bytes() { return (kTile * kTile + 3 * 16) * (int)sizeof(T); }
template <typename T> __device__ __forceinline__ int tile_at(int r, int c) {
    constexpr int N = VecTraits<T>::kVec;
    const int piece = c / N, block = c >> 5;
    const int moved = sizeof(T) == 4 ? piece ^ block ^ ((r & 1) << 2) : piece ^ (block >> 1) ^ ((r & 1) << 1);
    return (r * kTile + (r >> 5) * 16) * (int)sizeof(T) + moved * 16 + (c % N) * (int)sizeof(T);
}

struct MxTileMatrix {
    const void* x;
    uint8_t *data, *scales, *data_t, *scales_t;      // either pair may be NULL
    int64_t rows, cols;
    int tiles_x, tiles;
};
// One matrix or two (TWO): a training step's activations and weight in one launch share its last, partly filled round of CTAs
// (4100 x 2050 and 4010 x 2050 in bf16: 25.4 -> 20.6 us). One alone has its sizes in fixed places (29.7 against 31.5 us for 8192 x 5120).
struct MxTileParams {
    MxTileMatrix of[2];
    float* colsum;                                   // [ceil(rows / 128)][cols] of the first, or NULL
    int count;                                       // tiles of both
    template <bool TWO> __device__ __forceinline__ const MxTileMatrix& matrix(int& it) const {
        if constexpr (!TWO) return of[0];
        const bool second = it >= of[0].tiles;
        if (second) it -= of[0].tiles;
        return of[second];
    }
};

// One tile into shared memory, zeros outside the matrix, in asynchronous copies of 16 bytes or of 4 (rows that only allow
// that), which the caller commits and waits for, or (COPY 0) element by element.
template <typename T, int COPY, bool TWO>
__device__ __forceinline__ void mx4_fetch(const MxTileParams& both, uint8_t* tile, int it) {
    const MxTileMatrix& p = both.matrix<TWO>(it);
    constexpr int N = COPY > 0 ? COPY / (int)sizeof(T) : VecTraits<T>::kVec, kPacks = kTile / N;
    const int ty = it / p.tiles_x;
    const int64_t r0 = (int64_t)ty * kTile;
    const int c0 = (it - ty * p.tiles_x) * kTile;
    // a thread's column is the same in every round
    const int c = (int)(threadIdx.x % kPacks) * N, rows = (int)(p.rows - r0 < kTile ? p.rows - r0 : kTile), cols = (int)p.cols - c0;
    const T* src = (const T*)p.x + (r0 + threadIdx.x / kPacks) * p.cols + c0 + c;
    const int64_t step = (int64_t)(256 / kPacks) * p.cols;
#pragma unroll 8
    for (int r = threadIdx.x / kPacks; r < kTile; r += 256 / kPacks, src += step) {
        uint8_t* dst = tile + tile_at<T>(r, c);
        if constexpr (COPY > 0) {
            const bool in = r < rows && c < cols;
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
            if constexpr (COPY == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(in ? src : (const T*)p.x), "r"(in ? 16 : 0) : "memory");
            else
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(in ? src : (const T*)p.x), "r"(in ? 4 : 0) : "memory");
        } else {
            Pack<T, N> v;
#pragma unroll
            for (int j = 0; j < N; ++j) v.s[j] = r < rows && c + j < cols ? src[j] : from_f<T>(0.f);
            v.store(reinterpret_cast<T*>(dst));
        }
    }
}

// Thirty-two values (already multiplied by the factor, two at a time) as 16 bytes of codes; f(i) gives values i and i + 1.
template <typename F> __device__ __forceinline__ uint4 mx4_encode32(F&& f) {
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float u[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) { const float2 x = f(j * 8 + i); u[i] = x.x; u[i + 1] = x.y; }
        c[j] = mx4_encode8(u);
    }
    return make_uint4(c[0], c[1], c[2], c[3]);
}

template <typename T, int COPY, bool SUMS, bool TWO>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 1 : 3) k_mx4_tile(MxTileParams both) {
    extern __shared__ __align__(16) uint8_t tiles_smem[];
    __shared__ float sums[4][kTile];
    grid_dep_launch();
    grid_dep_wait();
    constexpr int N = VecTraits<T>::kVec, kWords = 32 * (int)sizeof(T) / 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int count = both.count;
    if constexpr (COPY > 0) {
        mx4_fetch<T, COPY, TWO>(both, tiles_smem, blockIdx.x);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    for (int it = blockIdx.x, buf = 0; it < count; it += gridDim.x, buf ^= COPY > 0 ? 1 : 0) {
        int at_tile = it;
        const MxTileMatrix& p = both.matrix<TWO>(at_tile);
        const int nb = (int)mx4_blocks(p.cols), tiles = (int)mx4_scale_tiles(p.cols), nbt = (int)mx4_blocks(p.rows), tiles_t = (int)mx4_scale_tiles(p.rows);
        const int ty = at_tile / p.tiles_x, tx = at_tile - ty * p.tiles_x;
        const int64_t r0 = (int64_t)ty * kTile;
        const int c0 = tx * kTile;
        uint8_t* tile = tiles_smem + buf * tile_bytes<T>();
        if constexpr (COPY > 0) {
            if (it + (int)gridDim.x < count) mx4_fetch<T, COPY, TWO>(both, tiles_smem + (buf ^ 1) * tile_bytes<T>(), it + gridDim.x);
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 1;" ::: "memory");
        } else {
            mx4_fetch<T, COPY, TWO>(both, tile, it);
        }
        __syncthreads();
        // the rows: a lane takes a block, a warp the four blocks of eight rows, twice
        if (p.data != nullptr) {
#pragma unroll 1
            for (int q = 0; q < 2; ++q) {
                const int tr = q * 64 + warp * 8 + (lane >> 2), blk = lane & 3;
                uint32_t w[kWords], m = 0u;
#pragma unroll
                for (int k = 0; k < kWords / 4; ++k) reinterpret_cast<uint4*>(w)[k] = *reinterpret_cast<const uint4*>(tile + tile_at<T>(tr, blk * 32 + k * N));
#pragma unroll
                for (int k = 0; k < kWords; ++k) m = amax_word<T>(m, w[k]);
                const uint32_t s = mx4_scale_byte(amax_bits<T>(m));
                const float f = mx4_factor(s);
                uint4 code = mx4_encode32([&](int i) {
                    float2 x;
                    if constexpr (sizeof(T) == 4) x = make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1]));
                    else x = word_values<T>(w[i / 2]);
                    mul2(x.x, x.y, f, f);
                    return x;
                });
                if (s == 255u) code = make_uint4(0u, 0u, 0u, 0u);
                const int64_t r = r0 + tr;
                if (tr < p.rows - r0) {
                    if (tx * 4 + blk < nb) *reinterpret_cast<uint4*>(p.data + (r * nb + tx * 4 + blk) * 16) = code;
                    p.scales[mx4_scale_word(r, tx, tiles) + blk] = (uint8_t)s;
                }
            }
        }
        // the columns: a thread takes two columns of a 32-row block; a warp 8 column pairs x the 4 blocks
        const int pair = warp * 8 + (lane & 7), blk = lane >> 3;
        uint32_t m[2] = {0u, 0u};
        uint32_t w[sizeof(T) == 4 ? 64 : 32];          // both columns, row by row
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint8_t* at = tile + tile_at<T>(blk * 32 + i, pair * 2);
            if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<uint2*>(&w[2 * i]) = *reinterpret_cast<const uint2*>(at);
                m[0] = amax_word<float>(m[0], w[2 * i]);
                m[1] = amax_word<float>(m[1], w[2 * i + 1]);
            } else {
                w[i] = *reinterpret_cast<const uint32_t*>(at);
                m[0] = amax_word<T>(m[0], w[i]);
            }
        }
        if constexpr (sizeof(T) == 2) {
            const float2 f = word_values<T>(m[0]);
            m[0] = __float_as_uint(f.x);
            m[1] = __float_as_uint(f.y);
        }
        const uint32_t s[2] = {mx4_scale_byte(m[0]), mx4_scale_byte(m[1])};
        const float f0 = mx4_factor(s[0]), f1 = mx4_factor(s[1]);
        uint32_t code[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float u[2][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float2 f;
                if constexpr (sizeof(T) == 4) f = make_float2(__uint_as_float(w[2 * (j * 8 + i)]), __uint_as_float(w[2 * (j * 8 + i) + 1]));
                else f = word_values<T>(w[j * 8 + i]);
                if constexpr (SUMS) { sum[0] += f.x; sum[1] += f.y; }
                mul2(f.x, f.y, f0, f1);
                u[0][i] = f.x;
                u[1][i] = f.y;
            }
            code[0][j] = mx4_encode8(u[0]);
            code[1][j] = mx4_encode8(u[1]);
        }
        if (p.data_t != nullptr) {
            const int b = ty * 4 + blk;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int c = c0 + pair * 2 + k;
                if (c < p.cols) {
                    const uint4 v = s[k] == 255u ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(code[k][0], code[k][1], code[k][2], code[k][3]);
                    if (b < nbt) *reinterpret_cast<uint4*>(p.data_t + ((int64_t)c * nbt + b) * 16) = v;
                    p.scales_t[mx4_scale_word(c, ty, tiles_t) + blk] = (uint8_t)s[k];
                }
            }
        }
        if constexpr (SUMS) {
            sums[blk][pair * 2] = sum[0];
            sums[blk][pair * 2 + 1] = sum[1];
            __syncthreads();
            if (threadIdx.x < kTile && c0 + (int)threadIdx.x < p.cols)
                both.colsum[ty * p.cols + c0 + threadIdx.x] =
                    (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
        }
        __syncthreads();          // the tile may be overwritten
    }
}

// The way of k_mx4_rows back: a warp takes four chunks of 256 values of a row, a lane eight codes of each. Rows that do not
// allow 16-byte stores go through shared memory, so that neighbouring lanes store neighbouring words (rows of an even number of
// bytes over 4) or elements.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                        int cols, MxWalk w) {
    grid_dep_launch();
    grid_dep_wait();
    __shared__ __align__(16) T turn[VEC ? 1 : 8][VEC ? 1 : kMxChunk];
    const int lane = threadIdx.x & 31;
    const int nb = (int)mx4_blocks(cols), tiles = (int)mx4_scale_tiles(cols);
    const bool words = sizeof(T) == 4 || (((reinterpret_cast<uintptr_t>(out) & 3u) == 0) && (cols & 1) == 0);
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
            constexpr int N = VecTraits<T>::kVec;
#pragma unroll
            for (int k = 0; k < 8 / N; ++k) {
                Pack<T, N> q;
#pragma unroll
                for (int i = 0; i < N; ++i) q.set(i, v[k * N + i]);
                if constexpr (VEC) { if (col + k * N < cols) q.store(o + k * N); }
                else q.store(&turn[threadIdx.x >> 5][lane * 8 + k * N]);
            }
            if constexpr (!VEC) {
                const T* mine = turn[threadIdx.x >> 5];
                T* start = o - lane * 8;
                const int left = cols - (col - lane * 8);          // values of the row from this chunk on
                __syncwarp();
                if (words) {
                    constexpr int M = 4 / (int)sizeof(T);
#pragma unroll
                    for (int i = 0; i < kMxChunk / M; i += 32)
                        if ((i + lane) * M < left) reinterpret_cast<uint32_t*>(start)[i + lane] = reinterpret_cast<const uint32_t*>(mine)[i + lane];
                } else {
#pragma unroll
                    for (int i = 0; i < kMxChunk; i += 32)
                        if (i + lane < left) start[i + lane] = mine[i + lane];
                }
                __syncwarp();
            }
        }
    }
}

template <typename T, int COPY, bool SUMS, bool TWO>
static int launch_tile(const MxTileParams& p, cudaStream_t st) {
    // two tiles of shared memory per CTA where the next one is on its way while a tile is encoded
    constexpr int smem = (COPY > 0 ? 2 : 1) * tile_bytes<T>();
    static PerDeviceOnce once;
    bool* set = once.slot();
    if (set == nullptr) return DC_ERR_LAUNCH;
    if (!*set) {
        if (cudaFuncSetAttribute(k_mx4_tile<T, COPY, SUMS, TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return check_launch();
        *set = true;
    }
    const int cap = sm_count() * (sizeof(T) == 4 ? 1 : 3);
    return launch_pdl(k_mx4_tile<T, COPY, SUMS, TWO>, dim3((unsigned)(p.count < cap ? p.count : cap)), dim3(256), smem, st, p);
}
template <typename T, bool SUMS, bool TWO = false>
static int launch_tile_copy(const MxTileParams& p, cudaStream_t st) {
    int access = row_access<T>(p.of[0].x, p.of[0].cols);
    if constexpr (TWO) {
        const int other = row_access<T>(p.of[1].x, p.of[1].cols);
        if (other < access) access = other;
    }
    if (access == 16) return launch_tile<T, 16, SUMS, TWO>(p, st);
    if constexpr (sizeof(T) == 2)
        if (access == 2) return launch_tile<T, 0, SUMS, TWO>(p, st);
    return launch_tile<T, 4, SUMS, TWO>(p, st);
}

static MxTileMatrix tile_matrix(const void* x, void* data, void* scales, void* data_t, void* scales_t, int64_t rows, int64_t cols) {
    const int64_t tx = divup64(cols, kTile), ty = divup64(rows, kTile);
    return MxTileMatrix{x, (uint8_t*)data, (uint8_t*)scales, (uint8_t*)data_t, (uint8_t*)scales_t, rows, cols, (int)tx, (int)(tx * ty)};
}

template <typename T>
static int quantize_t(const void* x, void* data, void* scales, void* data_t, void* scales_t, float* colsum, int64_t rows, int64_t cols, cudaStream_t st) {
    if (data_t == nullptr && colsum == nullptr) {
        const int segments = (int)divup64(mx4_scale_tiles(cols) * 128, kMxChunk * kMxAhead);
        int64_t ctas = divup64(rows * segments, 8);
        const int64_t cap = (int64_t)sm_count() * 5;
        if (ctas > cap) ctas = cap;
        const MxWalk w = mx_walk(rows, segments, ctas * 8);
        const dim3 grid((unsigned)ctas);
        const int access = row_access<T>(x, cols);
        if (access == 16) return launch_pdl(k_mx4_rows<T, 16>, grid, dim3(256), 0, st, (const T*)x, (uint8_t*)data, (uint8_t*)scales, (int)cols, w);
        if constexpr (sizeof(T) == 2)
            if (access == 2) return launch_pdl(k_mx4_rows<T, 2>, grid, dim3(256), 0, st, (const T*)x, (uint8_t*)data, (uint8_t*)scales, (int)cols, w);
        return launch_pdl(k_mx4_rows<T, 4>, grid, dim3(256), 0, st, (const T*)x, (uint8_t*)data, (uint8_t*)scales, (int)cols, w);
    }
    if (divup64(cols, kTile) * divup64(rows, kTile) > 0x3fffffffLL || rows > 0x7ffff000LL) return DC_ERR_SHAPE;
    MxTileParams p{{tile_matrix(x, data, scales, data_t, scales_t, rows, cols), MxTileMatrix{}}, colsum, 0};
    p.count = p.of[0].tiles;
    return colsum != nullptr ? launch_tile_copy<T, true>(p, st) : launch_tile_copy<T, false>(p, st);
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

// Both images of two matrices (checked as dc_mx4_quantize does) of one type in one launch.
int mx4_quantize_two(const void* x, void* data, void* scales, void* data_t, void* scales_t, int64_t rows, const void* x2, void* data2, void* scales2,
                     void* data_t2, void* scales_t2, int64_t rows2, int64_t cols, int dtype, cudaStream_t st) {
    if (divup64(cols, kTile) * (divup64(rows, kTile) + divup64(rows2, kTile)) > 0x3fffffffLL || rows > 0x7ffff000LL || rows2 > 0x7ffff000LL) return DC_ERR_SHAPE;
    MxTileParams p{{tile_matrix(x, data, scales, data_t, scales_t, rows, cols), tile_matrix(x2, data2, scales2, data_t2, scales_t2, rows2, cols)}, nullptr, 0};
    p.count = p.of[0].tiles + p.of[1].tiles;
    switch (dtype) {
        case DC_F32: return launch_tile_copy<float, false, true>(p, st);
        case DC_F16: return launch_tile_copy<__half, false, true>(p, st);
        default: return launch_tile_copy<__nv_bfloat16, false, true>(p, st);
    }
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
