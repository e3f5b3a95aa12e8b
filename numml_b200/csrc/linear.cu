// Dense product of the graph layers with its epilogue,  y = act(x w + bias) + residual,  and its gradients:
//   dz = dy act'(z),  dx = dz w^T,  dw = x^T dz,  dbias = column sums of dz
// with z = x w + bias as the forward pass left it.  x [m, k], w [k, n], y [m, n].
//
// This file holds the entry points, the products of few rows, those of double (the 5th-generation tensor
// instructions do not take it) and the passes around the products; linear_mma_kernel.cuh holds the products of the
// other types.
#include <cooperative_groups.h>

#include <type_traits>

#include "linear_mma.cuh"

namespace nb200 {
namespace {

constexpr int kTile = 64, kDepth = 16, kThreads = 256;

// ---- double: the double-precision tensor instruction (mma.sync, 16 x 8 x 8) ----------------------------------
// C[i, j] = sum_k A(i, k) B(k, j) on tiles of 64 rows x 32 WN columns, a warp per 32 x 32; blockIdx.z cuts the sum.
// A(i, k) is a[i * as + k] with A_K (k contiguous) or a[i + k * as]; B(k, j) is b[k + j * bs] with B_K or
// b[k * bs + j].  Sixteen terms of both operands are staged at a time, the next sixteen on their way in registers.
// Lines of 64 + 4 doubles: the sixteen lanes of a half-warp, four k by four rows, then touch sixteen banks.
// Measured: 65,536 x 128 -> 128 99 us = 21.8 TFLOP/s (the same on multiply-adds of 4 x 4 values per thread: 156 us, bound
// by shared-memory reads); latency of a step of sixteen terms bounds it, the library's product takes 76 us.
constexpr int kLine = 64 + 4;

__device__ __forceinline__ void mma_f64(double (&c)[4], const double (&a)[4], const double (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f64.f64.f64.f64 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+d"(c[0]), "+d"(c[1]), "+d"(c[2]), "+d"(c[3])
                 : "d"(a[0]), "d"(a[1]), "d"(a[2]), "d"(a[3]), "d"(b[0]), "d"(b[1]));
}

template <bool A_K, bool B_K, int ACT, int WN>
__global__ void __launch_bounds__(64 * WN, 4) double_kernel(int64_t rows, int64_t cols, int64_t depth, int64_t per,
                                                         const double* __restrict__ a, int64_t as, const double* __restrict__ b, int64_t bs,
                                                         Epilogue<double> ep) {
    constexpr int kBlock = 64 * WN, kCols = 32 * WN;
    constexpr int NA = kTile * kDepth / kBlock, NB = kCols * kDepth / kBlock;          // values per thread and step
    __shared__ double sa[2][kDepth][kLine], sb[2][kDepth][kLine];
    const int64_t i0 = blockIdx.x * int64_t(kTile), j0 = blockIdx.y * int64_t(kCols);
    const int t = threadIdx.x, lane = t % 32, g = lane / 4, q4 = lane % 4;
    const int wi = t / 32 % 2 * 32, wj = t / 64 * 32;                                  // the warp's corner in the tile
    const int64_t k_begin = blockIdx.z * per, k_end = min(depth, k_begin + per);
    double ra[NA], rb[NB];
    auto fetch = [&](int64_t k0) {
#pragma unroll
        for (int e = 0; e < NA; ++e) {
            const int x = t + e * kBlock, m = A_K ? x / kDepth : x % kTile, k = A_K ? x % kDepth : x / kTile;
            ra[e] = i0 + m < rows && k0 + k < k_end ? (A_K ? a[(i0 + m) * as + k0 + k] : a[i0 + m + (k0 + k) * as]) : 0.0;
        }
#pragma unroll
        for (int e = 0; e < NB; ++e) {
            const int x = t + e * kBlock, n = B_K ? x / kDepth : x % kCols, k = B_K ? x % kDepth : x / kCols;
            rb[e] = j0 + n < cols && k0 + k < k_end ? (B_K ? b[k0 + k + (j0 + n) * bs] : b[(k0 + k) * bs + j0 + n]) : 0.0;
        }
    };
    auto stage = [&](int s) {
#pragma unroll
        for (int e = 0; e < NA; ++e) {
            const int x = t + e * kBlock;
            sa[s][A_K ? x % kDepth : x / kTile][A_K ? x / kDepth : x % kTile] = ra[e];
        }
#pragma unroll
        for (int e = 0; e < NB; ++e) {
            const int x = t + e * kBlock;
            sb[s][B_K ? x % kDepth : x / kCols][B_K ? x / kDepth : x % kCols] = rb[e];
        }
    };
    double acc[2][4][4] = {};
    if (k_begin < k_end) {
        fetch(k_begin);
        stage(0);
    }
    __syncthreads();
    int s = 0;
    for (int64_t k0 = k_begin; k0 < k_end; k0 += kDepth, s ^= 1) {
        const bool more = k0 + kDepth < k_end;
        if (more) fetch(k0 + kDepth);
#pragma unroll
        for (int k = 0; k < kDepth; k += 8) {
            double af[2][4], bf[4][2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) af[u][r] = sa[s][k + q4 + (r / 2) * 4][wi + u * 16 + g + (r % 2) * 8];
#pragma unroll
            for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int r = 0; r < 2; ++r) bf[v][r] = sb[s][k + q4 + r * 4][wj + v * 8 + g];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) mma_f64(acc[u][v], af[u], bf[v]);
        }
        if (more) stage(s ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t i = i0 + wi + u * 16 + g + (r / 2) * 8, j = j0 + wj + v * 8 + q4 * 2 + r % 2;
                if (i >= rows || j >= cols) continue;
                double c = acc[u][v][r];
                if (ep.partial) {
                    ep.partial[(blockIdx.z * rows + i) * cols + j] = c;
                    continue;
                }
                if (ep.bias) c += ep.bias[j];
                if (ep.z) ep.z[i * cols + j] = c;
                c = activate<ACT>(c);
                if (ep.residual) c += ep.residual[i * ep.ldr + j];
                ep.y[i * cols + j] = c;
            }
}

// A product whose sum is empty (no input channels): act(bias) + residual.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) empty_sum_kernel(int64_t rows, int64_t cols, Epilogue<T> ep) {
    using A = acc_t<T>;
    for (int64_t e = blockIdx.x * int64_t(kThreads) + threadIdx.x; e < rows * cols; e += int64_t(gridDim.x) * kThreads) {
        const int64_t i = e / cols, j = e % cols;
        A v = ep.bias ? to_acc(ep.bias[j]) : A(0);
        if (ep.z) ep.z[e] = rounded_z<T, ACT>(v);
        v = activate<ACT>(v);
        if (ep.residual) v += to_acc(ep.residual[i * ep.ldr + j]);
        ep.y[e] = from_acc<T>(v);
    }
}

// Few rows (the features of a node or of a small graph): the call is the reading of w.  A block has kSkinnyCols columns and a
// share of the rows of w, eight columns to a thread, so that a warp reads lines of w; up to four rows of x go along.
// The blocks that share a column of blocks are a thread-block cluster and add their parts up through distributed
// shared memory in order of rank: one launch, no workspace, no atomics.
constexpr int kSkinnyCols = 64, kSkinnyRows = 4;

// When it is the faster way: it costs about 4 us and 0.36 us per million multiply-adds whatever the type, the tiles
// about 4 us and, for every 64 terms of the sum, 1.5 us (float), 0.28 us (16-bit), 5.4 us (double), as long as every
// tile has an SM to itself.  Measured, rows x 1024 x 1024: float 64 rows 26 us against 29, 96 rows 38 against 29;
// bfloat16 16 rows 8.1 against 8.5, 32 rows 14 against 8.5; double 64 rows 60 against 94, 128 rows 117 against 94.
// rows x 1024 x 64: float 256 rows 8 us against 29, bfloat16 7.9 against 8.5.
inline bool few_rows(int64_t rows, int64_t cols, size_t size) { return rows <= 512 && rows * cols <= (size == 2 ? 12 * 1024 : 48 * 1024); }

template <typename T, bool VECTOR, int ACT>
__global__ void __launch_bounds__(kThreads) skinny_kernel(int rows, int64_t cols, int64_t depth, int64_t share, const T* __restrict__ x,
                                                          int64_t ldx, const T* __restrict__ w, int64_t ldw, Epilogue<T> ep) {
    using A = acc_t<T>;
    constexpr int V = 8, kLanes = kSkinnyCols / V, kRowLanes = kThreads / kLanes, kWarps = kThreads / 32;
    __shared__ A part[kWarps][kSkinnyRows][kSkinnyCols];
    const unsigned rank = cooperative_groups::this_cluster().block_rank(), ranks = cooperative_groups::this_cluster().num_blocks();
    const int lane = threadIdx.x % kLanes, row_lane = threadIdx.x / kLanes;
    const int64_t j = blockIdx.x / ranks * int64_t(kSkinnyCols) + lane * V;
    const int i0 = blockIdx.y * kSkinnyRows, count = min(kSkinnyRows, rows - i0);
    const int64_t k_end = min(depth, (rank + 1) * share);
    A acc[kSkinnyRows][V] = {};
#pragma unroll 4
    for (int64_t k = rank * share + row_lane; k < k_end; k += kRowLanes) {
        A wv[V] = {};
        if (VECTOR) {
            constexpr int U = 16 / sizeof(T) < V ? 16 / sizeof(T) : V;
            if (j < cols)
#pragma unroll
                for (int q = 0; q < V; q += U) load_acc<T, U>(w + k * ldw + j + q, *reinterpret_cast<A(*)[U]>(wv + q));
        } else {
#pragma unroll
            for (int q = 0; q < V; ++q)
                if (j + q < cols) wv[q] = to_acc(w[k * ldw + j + q]);
        }
#pragma unroll
        for (int i = 0; i < kSkinnyRows; ++i) {
            if (i >= count) break;
            const A xv = to_acc(x[(i0 + i) * ldx + k]);
#pragma unroll
            for (int q = 0; q < V; ++q) acc[i][q] += xv * wv[q];
        }
    }
    // row lanes of a warp, then the warps, then the blocks
#pragma unroll
    for (int i = 0; i < kSkinnyRows; ++i)
#pragma unroll
        for (int q = 0; q < V; ++q) {
            A v = acc[i][q];
#pragma unroll
            for (int off = kLanes; off < 32; off <<= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
            if (threadIdx.x % 32 < kLanes) part[threadIdx.x / 32][i][lane * V + q] = v;
        }
    __syncthreads();
    A* sums = &part[0][0][0];
    for (int e = threadIdx.x; e < kSkinnyRows * kSkinnyCols; e += kThreads) {
        A v = sums[e];
        for (int q = 1; q < kWarps; ++q) v += sums[q * kSkinnyRows * kSkinnyCols + e];
        sums[e] = v;
    }
    auto cluster = cooperative_groups::this_cluster();
    cluster.sync();
    for (int e = rank * kThreads + threadIdx.x; e < kSkinnyRows * kSkinnyCols; e += ranks * kThreads) {
        const int i = i0 + e / kSkinnyCols;
        const int64_t col = blockIdx.x / ranks * int64_t(kSkinnyCols) + e % kSkinnyCols;
        if (i >= rows || col >= cols) continue;
        A v = 0;
        for (unsigned r = 0; r < ranks; ++r) v += *cluster.map_shared_rank(sums + e, r);
        if (ep.bias) v += to_acc(ep.bias[col]);
        if (ep.z) ep.z[i * cols + col] = rounded_z<T, ACT>(v);
        v = activate<ACT>(v);
        if (ep.residual) v += to_acc(ep.residual[i * ep.ldr + col]);
        ep.y[i * cols + col] = from_acc<T>(v);
    }
    cluster.sync();                                  // nobody leaves while its sums are being read
}

template <typename T, int ACT>
int skinny(int64_t rows, int64_t cols, int64_t depth, const T* x, int64_t ldx, const T* w, int64_t ldw, const Epilogue<T>& ep,
           cudaStream_t stream) {
    unsigned ranks = 1;                              // a share of at least 64 rows of w
    while (ranks < 8 && depth > int64_t(ranks) * 64) ranks *= 2;
    const int64_t blocks = ceil_div(cols, kSkinnyCols) * ranks;
    if (blocks > INT32_MAX) return NB200_ERR_TOO_LARGE;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(ceil_div(rows, kSkinnyRows)));
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim = {ranks, 1, 1};
    config.attrs = attribute;
    config.numAttrs = 1;
    const bool vector = cols % 8 == 0 && aligned16(w) && ldw * sizeof(T) % 16 == 0;
    const cudaError_t e = vector ? cudaLaunchKernelEx(&config, skinny_kernel<T, true, ACT>, static_cast<int>(rows), cols, depth,
                                                      ceil_div(depth, int64_t(ranks)), x, ldx, w, ldw, ep)
                                 : cudaLaunchKernelEx(&config, skinny_kernel<T, false, ACT>, static_cast<int>(rows), cols, depth,
                                                      ceil_div(depth, int64_t(ranks)), x, ldx, w, ldw, ep);
    return e == cudaSuccess ? launch_status() : NB200_ERR_CUDA;
}

// Sums over the leading index of partial [parts][size]: a block has 256 / lanes columns; lane l adds parts l, l + lanes,
// ..., then the lanes are added in order.  More lanes for more parts (4, 8 or 32), so that neither the loads of a
// lane follow one another for long nor lanes are idle.  The order depends on the sizes alone.  Up to two arrays in one
// launch.
template <typename T>
struct Join {
    int64_t size = 0;
    int parts = 0;
    const acc_t<T>* partial = nullptr;
    T* out = nullptr;
    __host__ __device__ int lanes() const { return parts <= 16 ? 4 : parts <= 64 ? 8 : 32; }
    int64_t blocks() const { return ceil_div(size, kThreads / lanes()); }
};
template <typename T>
__global__ void __launch_bounds__(kThreads) join_parts_kernel(Join<T> first, Join<T> second, unsigned first_blocks) {
    using A = acc_t<T>;
    __shared__ A sm[kThreads];
    const bool is_first = blockIdx.x < first_blocks;
    const Join<T>& j = is_first ? first : second;
    const int lanes = j.lanes(), columns = kThreads / lanes, lane = threadIdx.x / columns;
    const int64_t e = (blockIdx.x - (is_first ? 0 : first_blocks)) * int64_t(columns) + threadIdx.x % columns;
    A v = 0;
    if (e < j.size)
#pragma unroll 8
        for (int s = lane; s < j.parts; s += lanes) v += j.partial[s * j.size + e];
    sm[threadIdx.x] = v;
    __syncthreads();
    if (lane == 0 && e < j.size) {
#pragma unroll 4
        for (int q = 1; q < lanes; ++q) v += sm[q * columns + threadIdx.x];
        j.out[e] = from_acc<T>(v);
    }
}

// dz = dy act'(z) (not stored when dz is NULL: then dy is dz) and the column sums of dz over a band of rows.  dz is
// rounded to the type of the layer, which the products of 16-bit types need as their operand; its sums are of the unrounded.
// A thread owns V neighbouring columns of every row_lanes-th row; blockIdx.y selects the columns.  Moves
// 3 values per element (1 without an activation) and is bound by that: a million rows of 128 floats with silu 257 us =
// 6.3 TB/s, 0.96 of the copy rate; 131,072 x 512 bfloat16 93 us = 4.3 TB/s, where the slopes' instructions show.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) slope_kernel(int64_t rows, int64_t cols, int lanes, int64_t band, const T* __restrict__ dy,
                                                         int64_t ldd, const T* __restrict__ z, T* __restrict__ dz,
                                                         acc_t<T>* __restrict__ sums) {
    using A = acc_t<T>;
    __shared__ A sm[kThreads * V];
    const int lane = threadIdx.x % lanes, row_lane = threadIdx.x / lanes, row_lanes = kThreads / lanes;
    const int64_t j = (blockIdx.y * int64_t(lanes) + lane) * V;
    const bool live = row_lane < row_lanes && j < cols;
    const int64_t limit = min(rows, (blockIdx.x + 1) * band);
    A sum[V] = {};
    if (live) {
#pragma unroll 4
        for (int64_t i = blockIdx.x * band + row_lane; i < limit; i += row_lanes) {
            A v[V];
            load_acc<T, V>(dy + i * ldd + j, v);
            if (ACT != NB200_ACT_NONE) {
                A s[V];
                load_acc<T, V>(z + i * cols + j, s);
                slope_all<ACT>(s);
#pragma unroll
                for (int q = 0; q < V; ++q) v[q] *= s[q];
                store_acc<T, V>(dz + i * cols + j, v);
            }
#pragma unroll
            for (int q = 0; q < V; ++q) sum[q] += v[q];
        }
    }
    if (!sums) return;
#pragma unroll
    for (int q = 0; q < V; ++q) sm[threadIdx.x * V + q] = sum[q];
    __syncthreads();
    int width = 1;
    while (width < row_lanes) width <<= 1;
    for (int off = width >> 1; off > 0; off >>= 1) {
        const int other = threadIdx.x + off * lanes;
        if (live && row_lane < off && row_lane + off < row_lanes) {
#pragma unroll
            for (int q = 0; q < V; ++q) sm[threadIdx.x * V + q] = sum[q] += sm[other * V + q];
        }
        __syncthreads();
    }
    if (live && row_lane == 0)
#pragma unroll
        for (int q = 0; q < V; ++q) sums[blockIdx.x * cols + j + q] = sum[q];
}

// Bands of at least 32 rows, eight blocks per SM at most.
int64_t band_count(int64_t rows) {
    const int64_t wanted = ceil_div(rows, 32);
    return wanted < kSMs * 8 ? (wanted < 1 ? 1 : wanted) : kSMs * 8;
}

template <typename T, int V>
int slope_pass(int64_t m, int64_t n, int act, const T* dy, int64_t ldd, const T* z, T* dz, acc_t<T>* sums, cudaStream_t stream) {
    const int64_t vectors = n / V, lanes = vectors < kThreads ? vectors : kThreads, gy = ceil_div(vectors, lanes);
    if (gy > 65535) return NB200_ERR_TOO_LARGE;
    const int64_t bands = band_count(m);
    return NB200_DISPATCH_ACT(act, (slope_kernel<T, V, ACT><<<dim3(bands, gy), kThreads, 0, stream>>>(
                                        m, n, static_cast<int>(lanes), ceil_div(m, bands), dy, ldd, z, dz, sums), launch_status()));
}

template <typename T>
int join_parts(const Join<T>& first, const Join<T>& second, cudaStream_t stream) {
    const int64_t a = first.blocks(), b = second.blocks();
    if (a + b > INT32_MAX) return NB200_ERR_TOO_LARGE;
    if (a + b == 0) return NB200_OK;
    join_parts_kernel<T><<<static_cast<unsigned>(a + b), kThreads, 0, stream>>>(first, second, static_cast<unsigned>(a));
    return launch_status();
}

// Into how many parts the sum over the rows is cut for dw, so that there is work for every SM, and how long one is.
struct Split {
    int64_t parts, per;
};
Split split_sum(int64_t rows, int64_t cols, int64_t depth, int dtype) {
    if (rows == 0 || cols == 0 || depth == 0) return {1, kMmaChunk};
    if (dtype != NB200_F64) {
        const int64_t tiles = ceil_div(rows, kMmaTile) * ceil_div(cols, kMmaTile);
        const int64_t wanted = tiles < kSMs ? kSMs / tiles : 1;
        const int64_t per = ceil_div(ceil_div(depth, wanted), kMmaChunk) * kMmaChunk;
        return {ceil_div(depth, per), per};
    }
    const int64_t tiles = ceil_div(rows, kTile) * ceil_div(cols, kTile), wanted = ceil_div(kSMs * 4, tiles);
    const int64_t most = ceil_div(depth, 8 * kDepth);
    const int64_t parts = wanted < most ? wanted : (most < 1 ? 1 : most);
    const int64_t per = ceil_div(ceil_div(depth, parts), kDepth) * kDepth;
    return {ceil_div(depth, per), per};
}

size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }

struct BackwardLayout {
    size_t dz, sums, partial, total;
};
BackwardLayout backward_layout(int64_t m, int64_t k, int64_t n, int act, int dtype) {
    const size_t s = dense_dtype_size(dtype), a = dtype == NB200_F64 ? 8 : 4;
    BackwardLayout l;
    l.dz = 0;
    l.sums = l.dz + (act == NB200_ACT_NONE ? 0 : round16(s * m * n));
    l.partial = l.sums + round16(a * band_count(m) * n);
    l.total = l.partial + round16(a * split_sum(k, n, m, dtype).parts * k * n);
    return l;
}

template <typename T, bool A_K, bool B_K, int ACT>
int product(int64_t rows, int64_t cols, int64_t depth, Split split, const T* a, int64_t as, const T* b, int64_t bs,
            const Epilogue<T>& ep, int32_t* status, cudaStream_t stream) {
    if (depth == 0) {
        const int64_t blocks = ceil_div(rows * cols, kThreads);
        empty_sum_kernel<T, ACT><<<static_cast<unsigned>(blocks < kSMs * 8 ? blocks : kSMs * 8), kThreads, 0, stream>>>(rows, cols, ep);
        return launch_status();
    }
    if constexpr (!std::is_same<T, double>::value) {
        return mma_product<T, A_K, B_K, ACT>(rows, cols, depth, split.parts, split.per, a, as, b, bs, ep, status, stream);
    } else {
        const bool narrow = cols <= 32;
        const int64_t gx = ceil_div(rows, kTile), gy = ceil_div(cols, narrow ? 32 : 64);
        if (gx > INT32_MAX || gy > 65535 || split.parts > 65535) return NB200_ERR_TOO_LARGE;
        const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy), static_cast<unsigned>(split.parts));
        if (narrow)
            double_kernel<A_K, B_K, ACT, 1><<<grid, 64, 0, stream>>>(rows, cols, depth, split.per, a, as, b, bs, ep);
        else
            double_kernel<A_K, B_K, ACT, 2><<<grid, 128, 0, stream>>>(rows, cols, depth, split.per, a, as, b, bs, ep);
        return launch_status();
    }
}

Split whole(int64_t depth) { return {1, depth > 0 ? ceil_div(depth, kMmaChunk) * kMmaChunk : kMmaChunk}; }

template <typename T>
int backward(int64_t m, int64_t k, int64_t n, const T* dy, int64_t ldd, const T* x, int64_t ldx, const T* w, int64_t ldw, const T* z,
             int act, T* dx, T* dw, T* db, char* work, const BackwardLayout& lay, int dtype, int32_t* status, cudaStream_t stream) {
    using A = acc_t<T>;
    T* dz = act == NB200_ACT_NONE ? nullptr : reinterpret_cast<T*>(work + lay.dz);
    A* sums = reinterpret_cast<A*>(work + lay.sums);
    A* partial = reinterpret_cast<A*>(work + lay.partial);
    Join<T> join_db, join_dw;
    int rc = NB200_OK;
    if (dz || db) {
        constexpr int V = 16 / sizeof(T);
        const bool vector = n % V == 0 && ldd % V == 0 && aligned16(dy) && aligned16(z);
        rc = vector ? slope_pass<T, V>(m, n, act, dy, ldd, z, dz, db ? sums : nullptr, stream)
                    : slope_pass<T, 1>(m, n, act, dy, ldd, z, dz, db ? sums : nullptr, stream);
        if (rc != NB200_OK) return rc;
        if (db) join_db = Join<T>{n, static_cast<int>(band_count(m)), sums, db};
    }
    const T* g = dz ? dz : dy;
    const int64_t ldg = dz ? n : ldd;
    if (dx) {
        rc = product<T, true, true, NB200_ACT_NONE>(m, k, n, whole(n), g, ldg, w, ldw, {nullptr, nullptr, 0, nullptr, dx, nullptr}, status,
                                                    stream);
        if (rc != NB200_OK) return rc;
    }
    if (dw) {
        const Split split = split_sum(k, n, m, dtype);
        rc = product<T, false, false, NB200_ACT_NONE>(k, n, m, split, x, ldx, g, ldg, {nullptr, nullptr, 0, nullptr, nullptr, partial}, status,
                                                      stream);
        if (rc != NB200_OK) return rc;
        join_dw = Join<T>{k * n, static_cast<int>(split.parts), partial, dw};
    }
    return join_parts<T>(join_dw, join_db, stream);
}

bool bad_sizes(int64_t m, int64_t k, int64_t n) {
    constexpr int64_t most = int64_t(1) << 31;
    return m < 0 || k < 0 || n < 0 || m >= (int64_t(1) << 37) || k >= most || n >= most;
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" int nb200_linear_forward(int64_t m, int64_t k, int64_t n, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                    const void* bias, const void* residual, int64_t ldr, int activation, void* z, void* y,
                                    int32_t* status, int dtype, nb200_stream stream) {
    if (bad_sizes(m, k, n) || !known_dense_dtype(dtype) || !known_activation(activation)) return NB200_ERR_BAD_ARG;
    if (m == 0 || n == 0) return NB200_OK;
    if ((k > 0 && (!x || !w)) || !y || ldx < k || ldw < n || (residual && ldr < n)) return NB200_ERR_BAD_ARG;
    return NB200_DISPATCH_DENSE(dtype, ([&]() -> int {
        const Epilogue<T> ep{static_cast<const T*>(bias), static_cast<const T*>(residual), ldr, static_cast<T*>(z), static_cast<T*>(y), nullptr};
        if (few_rows(m, n, sizeof(T)))
            return NB200_DISPATCH_ACT(activation, (skinny<T, ACT>(m, n, k, static_cast<const T*>(x), ldx, static_cast<const T*>(w), ldw, ep,
                                                                  as_stream(stream))));
        return NB200_DISPATCH_ACT(activation, (product<T, true, false, ACT>(m, n, k, whole(k), static_cast<const T*>(x), ldx,
                                                                           static_cast<const T*>(w), ldw, ep, status, as_stream(stream))));
    }()));
}

extern "C" size_t nb200_linear_backward_workspace_bytes(int64_t m, int64_t k, int64_t n, int activation, int dtype) {
    if (bad_sizes(m, k, n) || !known_dense_dtype(dtype) || !known_activation(activation)) return 0;
    return backward_layout(m, k, n, activation, dtype).total;
}

extern "C" int nb200_linear_backward(int64_t m, int64_t k, int64_t n, const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                     const void* w, int64_t ldw, const void* z, int activation, void* dx, void* dw, void* dbias,
                                     void* work, size_t work_bytes, int32_t* status, int dtype, nb200_stream stream) {
    if (bad_sizes(m, k, n) || !known_dense_dtype(dtype) || !known_activation(activation)) return NB200_ERR_BAD_ARG;
    const size_t s = dense_dtype_size(dtype);
    const cudaStream_t st = as_stream(stream);
    if (m == 0 || n == 0) {                      // empty sums
        if ((dx && m * k > 0 && cudaMemsetAsync(dx, 0, s * m * k, st) != cudaSuccess) ||
            (dw && k * n > 0 && cudaMemsetAsync(dw, 0, s * k * n, st) != cudaSuccess) ||
            (dbias && n > 0 && cudaMemsetAsync(dbias, 0, s * n, st) != cudaSuccess))
            return NB200_ERR_CUDA;
        return NB200_OK;
    }
    if (!dy || lddy < n || ldx < k || ldw < n || (activation != NB200_ACT_NONE && !z)) return NB200_ERR_BAD_ARG;
    if (k > 0 && ((dx && !w) || (dw && !x))) return NB200_ERR_BAD_ARG;
    const BackwardLayout lay = backward_layout(m, k, n, activation, dtype);
    if (lay.total > 0 && (!work || work_bytes < lay.total)) return NB200_ERR_WORKSPACE;
    if (!aligned16(work)) return NB200_ERR_ALIGN;
    return NB200_DISPATCH_DENSE(dtype, (backward<T>(m, k, n, static_cast<const T*>(dy), lddy, static_cast<const T*>(x), ldx,
                                                    static_cast<const T*>(w), ldw, static_cast<const T*>(z), activation,
                                                    k > 0 ? static_cast<T*>(dx) : nullptr, k > 0 ? static_cast<T*>(dw) : nullptr,
                                                    static_cast<T*>(dbias), static_cast<char*>(work), lay, dtype, status, st)));
}
