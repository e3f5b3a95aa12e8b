// Group norm with an activation over channels-last rows [rows, channels]:
//   y = act(xhat * gamma + beta),   xhat = (x - mean) * rstd,   rstd = (var + eps)^(-1/2)
// where mean and (biased) variance are taken over the rows of a segment (one graph of a batch) and the
// channels / groups neighbouring channels of a group.  Backward, with dz = dy act'(z) and h = dz gamma:
//   dx = rstd (h - mean(h) - xhat mean(h xhat)),  dgamma = sum dz xhat,  dbeta = sum dz.
//
// Segments may be of any length, so rows are cut into equal chunks, one per block, and not by segment: every block
// has as many rows as the others, however ragged the batch is.  (A chunk's pieces come one after the other, though, at
// about 0.6 us each: hundreds of segments of a row or two side by side are slow where the kernels of short segments
// below do not take them.)  A chunk holds pieces of several segments and a segment pieces of several chunks; piece
// (block b, segment s) has workspace slot b + s, which is unique because b and s never decrease from one piece to the
// next.  A pass writes per-channel partial results of its pieces, a small kernel joins them per (segment, group) in a
// fixed order (no atomics: two runs give the same bits), and a second pass over the rows applies them.
//
// Variances come from differences: a thread sums (x - k) and (x - k)^2 with k the first value it meets
// of its channel in the piece, and partial results are joined as (count, mean, sum of squared
// deviations), the join over pieces in 64 bits.  E[x^2] - E[x]^2 never appears.
//
// Measured on a million rows of 128 floats in 32 groups, silu (537 MB an array; copy 6548 GB/s): stats 104 us = 5.2 TB/s,
// apply 173 us = 6.2, gradient sums 204 us = 5.3, gradient 265 us = 6.1, joins 6-10 us each: bound by memory.  An array
// that does not fit on chip is read twice in each direction.
#include <cooperative_groups.h>

#include <type_traits>

#include "dense_common.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 256;

// Everything that the kernels of a call share.
struct Shape {
    int64_t rows, chunk;          // rows of the array; rows per block
    int channels, groups, lanes;  // lanes = vectors of a row that a block covers (blockIdx.y selects which)
    int64_t segments;
    const int64_t* ptr;           // segments + 1 row pointers, or NULL: segments of `equal` rows
    int64_t equal;
    int64_t handed;               // 0, or: segments of more rows than this are left to handed_*_kernel
};

__device__ __forceinline__ int64_t clamp_row(int64_t r, int64_t rows) { return r < 0 ? 0 : (r > rows ? rows : r); }
__device__ __forceinline__ int64_t segment_begin(const Shape& sh, int64_t s) {
    return sh.ptr ? clamp_row(sh.ptr[s], sh.rows) : s * sh.equal;
}

// The segment that holds `row` (-1: before the first, `segments`: behind the last) and where the run of
// rows with that answer ends.  Row pointers out of order or out of range give some in-range answer that
// still advances, so a broken pointer array cannot make a kernel leave its arrays or loop for ever.
__device__ __forceinline__ int64_t find_segment(const Shape& sh, int64_t row, int64_t limit, int64_t& end) {
    if (!sh.ptr) {
        const int64_t s = row / sh.equal;
        end = min(limit, (s + 1) * sh.equal);
        return s;
    }
    int64_t lo = 0, hi = sh.segments + 1;          // first index whose pointer is > row
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (sh.ptr[mid] > row) hi = mid; else lo = mid + 1;
    }
    end = lo <= sh.segments ? min(limit, max(sh.ptr[lo], row + 1)) : limit;
    return lo - 1;
}

// The pieces of a block's chunk of rows, one after the other: piece(s, slot, row, end) for rows of segment s, whose partial
// results have that place in the workspace, outside(row, end) for rows of no segment.
struct ChunkPieces {
    const Shape& sh;
    template <typename Piece, typename Outside>
    __device__ __forceinline__ void each(Piece&& piece, Outside&& outside) const {
        const int64_t limit = min(sh.rows, (blockIdx.x + 1) * sh.chunk);
        for (int64_t row = blockIdx.x * sh.chunk, end; row < limit; row = end) {
            const int64_t s = find_segment(sh, row, limit, end);
            if (s < 0 || s >= sh.segments) outside(row, end);
            else piece(s, blockIdx.x + s, row, end);
        }
    }
};

// The segments of more than sh.handed rows as an array of their own: they follow one another in it, and each block of the
// grid has an equal run of its rows.  There are at most kMostHanded (the host sees to that; of broken row pointers some are
// left out).  Among few segments a block looks at all of them (512: 2.3 us a launch that finds none); among more it
// searches: each long segment holds a row whose number is a multiple of sh.handed, so there are rows / sh.handed searches
// (3.8 us), however many segments there are.
constexpr int kMostHanded = 72, kFewSegments = 2048;
struct HandedPieces {
    int count;
    int segment[kMostHanded];
    int64_t start[kMostHanded + 1];      // where a segment starts in that array
    int64_t begin[kMostHanded];          // and among all rows
    int found[kMostHanded];

    __device__ void find(const Shape& sh) {              // this object is in shared memory; all threads of the block
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        auto add = [&](int64_t s) {
            const int q = atomicAdd(&count, 1);
            if (q < kMostHanded) found[q] = static_cast<int>(s);
        };
        const int64_t row = threadIdx.x * sh.handed;
        if (sh.segments <= kFewSegments) {
            for (int64_t s = threadIdx.x; s < sh.segments; s += kThreads)
                if (segment_begin(sh, s + 1) - segment_begin(sh, s) > sh.handed) add(s);
        } else if (threadIdx.x < kMostHanded && row < sh.rows) {
            int64_t end;
            const int64_t s = find_segment(sh, row, sh.rows, end);
            if (s >= 0 && s < sh.segments) {
                const int64_t first = segment_begin(sh, s);          // a segment that holds an earlier such row has been found there
                if (segment_begin(sh, s + 1) - first > sh.handed && (row == 0 || first > row - sh.handed)) add(s);
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) count = min(count, kMostHanded);
        __syncthreads();
        if (threadIdx.x < count) {                       // in ascending order, whoever came first
            int rank = 0;
            for (int q = 0; q < count; ++q)
                rank += found[q] < found[threadIdx.x] || (found[q] == found[threadIdx.x] && q < threadIdx.x);
            segment[rank] = found[threadIdx.x];
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            start[0] = 0;
            for (int q = 0; q < count; ++q) {
                begin[q] = segment_begin(sh, segment[q]);
                start[q + 1] = start[q] + max(int64_t(0), segment_begin(sh, segment[q] + 1) - begin[q]);
            }
        }
        __syncthreads();
    }
    __device__ __forceinline__ int64_t chunk() const { return (start[count] + gridDim.x - 1) / gridDim.x; }
    template <typename Piece, typename Outside>
    __device__ __forceinline__ void each(Piece&& piece, Outside&&) const {
        const int64_t first = blockIdx.x * chunk(), limit = min(first + chunk(), start[count]);
        for (int q = 0; q < count; ++q) {
            const int64_t row = max(first, start[q]), end = min(limit, start[q + 1]);
            if (row < end) piece(int64_t(segment[q]), int64_t(blockIdx.x) + q, row - start[q] + begin[q], end - start[q] + begin[q]);
        }
    }
};

// Join (n, mean, m2) with (nb, mean_b, m2_b).
template <typename A>
__device__ __forceinline__ void join(A& n, A& mean, A& m2, A nb, A mean_b, A m2_b) {
    if (nb == A(0)) return;
    if (n == A(0)) {
        n = nb;
        mean = mean_b;
        m2 = m2_b;
        return;
    }
    const A total = n + nb;
    const A d = mean_b - mean, f = nb / total;
    mean += d * f;
    m2 += m2_b + d * d * n * f;
    n = total;
}

// ---- forward, first pass: per channel (mean, m2) of every piece ---------------------------------------
template <typename T, int V, typename Pieces>
__device__ __forceinline__ void form_stats(const Shape& sh, const Pieces& pieces, const T* __restrict__ x, acc_t<T>* __restrict__ part) {
    using A = acc_t<T>;
    __shared__ A sm_mean[kThreads * V], sm_m2[kThreads * V], sm_n[kThreads];
    const int lane = threadIdx.x % sh.lanes, row_lane = threadIdx.x / sh.lanes, row_lanes = kThreads / sh.lanes;
    const int c = (blockIdx.y * sh.lanes + lane) * V;
    const bool live = row_lane < row_lanes && c < sh.channels;
    pieces.each([&](int64_t, int64_t slot, int64_t row, int64_t end) {
        A k[V] = {}, sum[V] = {}, sq[V] = {}, n = 0;
        if (live) {
            int64_t r = row + row_lane;
            if (r < end) load_acc<T, V>(x + r * sh.channels + c, k);
            n = static_cast<A>(r < end ? (end - r + row_lanes - 1) / row_lanes : 0);
#pragma unroll 8
            for (; r < end; r += row_lanes) {
                A v[V];
                load_acc<T, V>(x + r * sh.channels + c, v);
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    const A d = v[q] - k[q];
                    sum[q] += d;
                    sq[q] += d * d;
                }
            }
        }
        A mean[V], m2[V];
#pragma unroll
        for (int q = 0; q < V; ++q) {
            const A d = n > A(0) ? sum[q] / n : A(0);
            mean[q] = k[q] + d;
            m2[q] = max(sq[q] - d * sum[q], A(0));
            if (sq[q] != sq[q]) m2[q] = sq[q];      // NaN must not end as zero
            sm_mean[threadIdx.x * V + q] = mean[q];
            sm_m2[threadIdx.x * V + q] = m2[q];
        }
        sm_n[threadIdx.x] = n;
        __syncthreads();
        int width = 1;
        while (width < row_lanes) width <<= 1;
        for (int off = width >> 1; off > 0; off >>= 1) {
            const int other = threadIdx.x + off * sh.lanes;
            if (live && row_lane < off && row_lane + off < row_lanes) {
                const A nb = sm_n[other];
                A n_new = n;
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    n_new = n;
                    join(n_new, mean[q], m2[q], nb, sm_mean[other * V + q], sm_m2[other * V + q]);
                    sm_mean[threadIdx.x * V + q] = mean[q];
                    sm_m2[threadIdx.x * V + q] = m2[q];
                }
                n = n_new;
                sm_n[threadIdx.x] = n;
            }
            __syncthreads();
        }
        if (live && row_lane == 0) {
            A* out = part + slot * 2 * sh.channels + c;
#pragma unroll
            for (int q = 0; q < V; ++q) {
                out[q] = mean[q];
                out[sh.channels + q] = m2[q];
            }
        }
    }, [](int64_t, int64_t) {});
}
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) stats_kernel(Shape sh, const T* __restrict__ x, acc_t<T>* __restrict__ part) {
    form_stats<T, V>(sh, ChunkPieces{sh}, x, part);
}

// Rows of segment s that lie in chunk b.
__device__ __forceinline__ int64_t piece_rows(int64_t begin, int64_t end, int64_t b, int64_t chunk) {
    return min(end, (b + 1) * chunk) - max(begin, b * chunk);
}

// One team of TEAM threads per (segment, group): the mean from the pieces' means weighted by their entries, then the
// sum of squared deviations from it, sum of m2 + entries (piece's mean - mean)^2, all in 64 bits.
template <int TEAM>
__device__ __forceinline__ double team_sum(double v, double* sm) {
    const int t = threadIdx.x % TEAM;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
    if (TEAM == 32) return v;
    __syncthreads();
    if (t % 32 == 0) sm[t / 32] = v;
    __syncthreads();
    double total = 0;
#pragma unroll
    for (int q = 0; q < TEAM / 32; ++q) total += sm[q];
    return total;
}

constexpr int join_threads(int team) { return team < kThreads ? kThreads : team; }

// A segment's pieces: rows begin .. end of the array that chunks of `chunk` rows cut up, the first piece in slot `slot`.
struct Span {
    int64_t begin, end, chunk;
    __device__ __forceinline__ int64_t first() const { return begin / chunk; }
    __device__ __forceinline__ int64_t pieces() const { return end > begin ? (end - 1) / chunk - first() + 1 : 0; }
};
__device__ __forceinline__ Span segment_span(const Shape& sh, int64_t s) {
    const int64_t begin = segment_begin(sh, s);
    return {begin, max(begin, segment_begin(sh, s + 1)), sh.chunk};
}

template <typename A, int TEAM>
__device__ __forceinline__ void join_stats(const Span& span, bool live, const A* base, int channels, int width, double eps,
                                           double* sm, A* mean_out, A* rstd_out) {
    const int t = threadIdx.x % TEAM;
    const int64_t first = span.first(), pieces = live ? span.pieces() : 0;
    // the team's threads go along the channels first; what does not divide is idle
    const int per = width < TEAM ? width : TEAM, lanes = TEAM / per, lane = t / per;
    double sum = 0;
    for (int c = t % per; c < width; c += per)
        if (lane < lanes)
#pragma unroll 4
            for (int64_t b = lane; b < pieces; b += lanes)
                sum += static_cast<double>(piece_rows(span.begin, span.end, first + b, span.chunk)) * static_cast<double>(base[b * 2 * channels + c]);
    const double n = static_cast<double>(span.end - span.begin) * width;
    const double mean = team_sum<TEAM>(sum, sm) / (n > 0 ? n : 1.0);
    double m2 = 0;
    for (int c = t % per; c < width; c += per)
        if (lane < lanes)
#pragma unroll 4
            for (int64_t b = lane; b < pieces; b += lanes) {
                const A* p = base + b * 2 * channels + c;
                const double d = static_cast<double>(p[0]) - mean;
                m2 += static_cast<double>(p[channels]) + static_cast<double>(piece_rows(span.begin, span.end, first + b, span.chunk)) * d * d;
            }
    m2 = team_sum<TEAM>(m2, sm);
    if (live && t == 0) {
        *mean_out = static_cast<A>(n > 0 ? mean : 0.0);
        *rstd_out = n > 0 ? static_cast<A>(1.0 / sqrt(m2 / n + eps)) : A(0);
    }
}

template <typename A, int TEAM>
__global__ void __launch_bounds__(join_threads(TEAM)) stats_join_kernel(Shape sh, const A* __restrict__ part, double eps,
                                                              A* __restrict__ mean_out, A* __restrict__ rstd_out) {
    __shared__ double sm[join_threads(TEAM) / 32];
    const int64_t item = blockIdx.x * int64_t(join_threads(TEAM) / TEAM) + threadIdx.x / TEAM;
    const bool live = item < sh.segments * sh.groups;
    const int64_t s = live ? item / sh.groups : 0;
    const int g = static_cast<int>(live ? item % sh.groups : 0), width = sh.channels / sh.groups;
    const Span span = segment_span(sh, s);
    join_stats<A, TEAM>(span, live, part + (span.first() + s) * 2 * sh.channels + g * width, sh.channels, width, eps, sm, mean_out + item,
                        rstd_out + item);
}

// ---- what a thread knows of its V channels ------------------------------------------------------------
template <typename T, int V>
struct ChannelParams {
    acc_t<T> gamma[V], beta[V];
    int group[V];
    __device__ __forceinline__ void load(const Shape& sh, int c, const T* w, const T* b) {
        const int width = sh.channels / sh.groups;
#pragma unroll
        for (int q = 0; q < V; ++q) {
            gamma[q] = w ? to_acc(w[c + q]) : acc_t<T>(1);
            beta[q] = b ? to_acc(b[c + q]) : acc_t<T>(0);
            group[q] = (c + q) / width;
        }
    }
};

// The statistics may be this launch's own results: no __restrict__.
template <typename T, int V, int ACT, typename Pieces>
__device__ __forceinline__ void apply_rows(const Shape& sh, const Pieces& pieces, const T* __restrict__ x, const T* __restrict__ w,
                                           const T* __restrict__ bias, const acc_t<T>* mean, const acc_t<T>* rstd, T* __restrict__ y) {
    using A = acc_t<T>;
    const int lane = threadIdx.x % sh.lanes, row_lane = threadIdx.x / sh.lanes, row_lanes = kThreads / sh.lanes;
    const int c = (blockIdx.y * sh.lanes + lane) * V;
    if (row_lane >= row_lanes || c >= sh.channels) return;
    ChannelParams<T, V> cp;
    cp.load(sh, c, w, bias);
    pieces.each([&](int64_t s, int64_t, int64_t row, int64_t end) {
        A m[V], a[V];
#pragma unroll
        for (int q = 0; q < V; ++q) {
            m[q] = mean[s * sh.groups + cp.group[q]];
            a[q] = rstd[s * sh.groups + cp.group[q]] * cp.gamma[q];
        }
#pragma unroll 4
        for (int64_t r = row + row_lane; r < end; r += row_lanes) {
            A v[V];
            load_acc<T, V>(x + r * sh.channels + c, v);
#pragma unroll
            for (int q = 0; q < V; ++q) v[q] = (v[q] - m[q]) * a[q] + cp.beta[q];
            activate_all<ACT>(v);
            store_acc<T, V>(y + r * sh.channels + c, v);
        }
    }, [&](int64_t row, int64_t end) {
        const A zero[V] = {};
        for (int64_t r = row + row_lane; r < end; r += row_lanes) store_acc<T, V>(y + r * sh.channels + c, zero);
    });
}
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) apply_kernel(Shape sh, const T* __restrict__ x, const T* __restrict__ w,
                                                         const T* __restrict__ bias, const acc_t<T>* __restrict__ mean,
                                                         const acc_t<T>* __restrict__ rstd, T* __restrict__ y) {
    apply_rows<T, V, ACT>(sh, ChunkPieces{sh}, x, w, bias, mean, rstd, y);
}

// Both passes over the segments that short_forward_kernel has handed over, in one cooperative launch; it finds out for
// itself whether there are any, and is done when there are none.  sh.ptr is what that kernel has kept of the row pointers.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, 2) handed_forward_kernel(Shape sh, const T* __restrict__ x, const T* __restrict__ w,
                                                                     const T* __restrict__ bias, double eps, acc_t<T>* mean, acc_t<T>* rstd,
                                                                     acc_t<T>* part, T* __restrict__ y) {
    using A = acc_t<T>;
    __shared__ HandedPieces pieces;
    __shared__ double sm[kThreads / 32];
    pieces.find(sh);
    if (pieces.count == 0) return;                       // the same for all blocks
    form_stats<T, V>(sh, pieces, x, part);
    cooperative_groups::this_grid().sync();
    const int width = sh.channels / sh.groups, n = pieces.count * sh.groups;
    for (int item = blockIdx.y * gridDim.x + blockIdx.x; item < n; item += gridDim.x * gridDim.y) {
        const int q = item / sh.groups, g = item % sh.groups;
        const Span span{pieces.start[q], pieces.start[q + 1], pieces.chunk()};
        const int64_t to = int64_t(pieces.segment[q]) * sh.groups + g;
        join_stats<A, kThreads>(span, true, part + (span.first() + q) * 2 * sh.channels + g * width, sh.channels, width, eps, sm, mean + to,
                                rstd + to);
    }
    cooperative_groups::this_grid().sync();
    apply_rows<T, V, ACT>(sh, pieces, x, w, bias, mean, rstd, y);
}

// ---- backward, first pass: per channel (sum dz, sum dz xhat) of every piece and of every block ---------
template <typename T, int V, int ACT, typename Pieces>
__device__ __forceinline__ void form_grad_sums(const Shape& sh, const Pieces& pieces, const T* __restrict__ x, const T* __restrict__ dy,
                                               const T* __restrict__ w, const T* __restrict__ bias, const acc_t<T>* __restrict__ mean,
                                               const acc_t<T>* __restrict__ rstd, acc_t<T>* part, acc_t<T>* block_sums) {
    using A = acc_t<T>;
    __shared__ A sm[2][kThreads * V];
    const int lane = threadIdx.x % sh.lanes, row_lane = threadIdx.x / sh.lanes, row_lanes = kThreads / sh.lanes;
    const int c = (blockIdx.y * sh.lanes + lane) * V;
    const bool live = row_lane < row_lanes && c < sh.channels;
    ChannelParams<T, V> cp;
    if (live) cp.load(sh, c, w, bias);
    A total1[V] = {}, total2[V] = {};
    pieces.each([&](int64_t s, int64_t slot, int64_t row, int64_t end) {
        A s1[V] = {}, s2[V] = {};
        if (live) {
            A m[V], rs[V];
#pragma unroll
            for (int q = 0; q < V; ++q) {
                m[q] = mean[s * sh.groups + cp.group[q]];
                rs[q] = rstd[s * sh.groups + cp.group[q]];
            }
#pragma unroll 4
            for (int64_t r = row + row_lane; r < end; r += row_lanes) {
                A v[V], g[V];
                load_acc<T, V>(x + r * sh.channels + c, v);
                load_acc<T, V>(dy + r * sh.channels + c, g);
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    const A xhat = (v[q] - m[q]) * rs[q];
                    const A dz = g[q] * activate_slope<ACT>(xhat * cp.gamma[q] + cp.beta[q]);
                    s1[q] += dz;
                    s2[q] += dz * xhat;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < V; ++q) {
            sm[0][threadIdx.x * V + q] = s1[q];
            sm[1][threadIdx.x * V + q] = s2[q];
        }
        __syncthreads();
        int width = 1;
        while (width < row_lanes) width <<= 1;
        for (int off = width >> 1; off > 0; off >>= 1) {
            const int other = threadIdx.x + off * sh.lanes;
            if (live && row_lane < off && row_lane + off < row_lanes) {
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    sm[0][threadIdx.x * V + q] = s1[q] += sm[0][other * V + q];
                    sm[1][threadIdx.x * V + q] = s2[q] += sm[1][other * V + q];
                }
            }
            __syncthreads();
        }
        if (live && row_lane == 0) {
            A* out = part + slot * 2 * sh.channels + c;
#pragma unroll
            for (int q = 0; q < V; ++q) {
                out[q] = s1[q];
                out[sh.channels + q] = s2[q];
                total1[q] += s1[q];
                total2[q] += s2[q];
            }
        }
    }, [](int64_t, int64_t) {});
    if (live && row_lane == 0) {
        A* out = block_sums + blockIdx.x * int64_t(2) * sh.channels + c;
#pragma unroll
        for (int q = 0; q < V; ++q) {
            out[q] = total1[q];
            out[sh.channels + q] = total2[q];
        }
    }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) grad_sums_kernel(Shape sh, const T* __restrict__ x, const T* __restrict__ dy,
                                                             const T* __restrict__ w, const T* __restrict__ bias,
                                                             const acc_t<T>* __restrict__ mean, const acc_t<T>* __restrict__ rstd,
                                                             acc_t<T>* __restrict__ part, acc_t<T>* __restrict__ block_sums) {
    form_grad_sums<T, V, ACT>(sh, ChunkPieces{sh}, x, dy, w, bias, mean, rstd, part, block_sums);
}

// mean(h) and mean(h xhat) of a (segment, group), from the per-channel sums of its pieces.
template <typename T, int TEAM>
__device__ __forceinline__ void join_grads(const Span& span, bool live, const acc_t<T>* base, int channels, int width,
                                           const T* __restrict__ w, double* sm, acc_t<T>* coef) {
    const int t = threadIdx.x % TEAM;
    const int64_t pieces = live ? span.pieces() : 0;
    const int per = width < TEAM ? width : TEAM, lanes = TEAM / per, lane = t / per;
    double a = 0, b = 0;
    for (int c = t % per; c < width; c += per) {
        double ca = 0, cb = 0;
        if (lane < lanes)
#pragma unroll 4
            for (int64_t q = lane; q < pieces; q += lanes) {
                const acc_t<T>* p = base + q * 2 * channels + c;
                ca += static_cast<double>(p[0]);
                cb += static_cast<double>(p[channels]);
            }
        const double gamma = w ? static_cast<double>(to_acc(w[c])) : 1.0;
        a += gamma * ca;
        b += gamma * cb;
    }
    a = team_sum<TEAM>(a, sm);
    b = team_sum<TEAM>(b, sm);
    if (live && t == 0) {
        const double n = static_cast<double>(span.end - span.begin) * width;
        coef[0] = static_cast<acc_t<T>>(n > 0 ? a / n : 0.0);
        coef[1] = static_cast<acc_t<T>>(n > 0 ? b / n : 0.0);
    }
}

template <typename T, int TEAM>
__global__ void __launch_bounds__(join_threads(TEAM)) grad_join_kernel(Shape sh, const acc_t<T>* __restrict__ part, const T* __restrict__ w,
                                                             acc_t<T>* __restrict__ coef) {
    __shared__ double sm[join_threads(TEAM) / 32];
    const int64_t item = blockIdx.x * int64_t(join_threads(TEAM) / TEAM) + threadIdx.x / TEAM;
    const bool live = item < sh.segments * sh.groups;
    const int64_t s = live ? item / sh.groups : 0;
    const int g = static_cast<int>(live ? item % sh.groups : 0), width = sh.channels / sh.groups;
    const Span span = segment_span(sh, s);
    join_grads<T, TEAM>(span, live, part + (span.first() + s) * 2 * sh.channels + g * width, sh.channels, width, w ? w + g * width : nullptr, sm,
                        coef + 2 * item);
}

// dbeta and dgamma: columns of sums [parts][2][channels] added up; 32 columns x 32 lanes of a block, in an order
// that depends on the sizes alone.
template <typename T>
__global__ void __launch_bounds__(1024) column_sums_kernel(int64_t parts, int channels, const acc_t<T>* __restrict__ sums,
                                                           T* __restrict__ dbeta, T* __restrict__ dgamma) {
    __shared__ double sm[32][33];
    const int col = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
    double a = 0;
    if (col < 2 * channels)
#pragma unroll 8
        for (int64_t b = lane; b < parts; b += 32) a += static_cast<double>(sums[b * 2 * channels + col]);
    sm[lane][threadIdx.x % 32] = a;
    __syncthreads();
    // transposed, so that a warp adds the 32 lanes of one column
    a = sm[threadIdx.x % 32][lane];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) a += __shfl_xor_sync(0xFFFFFFFFu, a, off);
    const int mine = blockIdx.x * 32 + lane;
    if (threadIdx.x % 32 == 0 && mine < 2 * channels) {
        T* out = mine < channels ? dbeta : dgamma;
        if (out) out[mine % channels] = from_acc<T>(static_cast<acc_t<T>>(a));
    }
}

template <typename T, int V, int ACT, typename Pieces>
__device__ __forceinline__ void apply_grads(const Shape& sh, const Pieces& pieces, const T* __restrict__ x, const T* __restrict__ dy,
                                            const T* __restrict__ w, const T* __restrict__ bias, const acc_t<T>* __restrict__ mean,
                                            const acc_t<T>* __restrict__ rstd, const acc_t<T>* coef, T* __restrict__ dx) {
    using A = acc_t<T>;
    const int lane = threadIdx.x % sh.lanes, row_lane = threadIdx.x / sh.lanes, row_lanes = kThreads / sh.lanes;
    const int c = (blockIdx.y * sh.lanes + lane) * V;
    if (row_lane >= row_lanes || c >= sh.channels) return;
    ChannelParams<T, V> cp;
    cp.load(sh, c, w, bias);
    pieces.each([&](int64_t s, int64_t, int64_t row, int64_t end) {
        A m[V], rs[V], c1[V], c2[V];
#pragma unroll
        for (int q = 0; q < V; ++q) {
            const int64_t item = s * sh.groups + cp.group[q];
            m[q] = mean[item];
            rs[q] = rstd[item];
            c1[q] = coef[2 * item];
            c2[q] = coef[2 * item + 1];
        }
        // backwards: what the first pass read last is still in L2
#pragma unroll 4
        for (int64_t r = end - 1 - row_lane; r >= row; r -= row_lanes) {
            A v[V], g[V];
            load_acc<T, V>(x + r * sh.channels + c, v);
            load_acc<T, V>(dy + r * sh.channels + c, g);
            A slope[V];
#pragma unroll
            for (int q = 0; q < V; ++q) {
                v[q] = (v[q] - m[q]) * rs[q];
                slope[q] = v[q] * cp.gamma[q] + cp.beta[q];
            }
            slope_all<ACT>(slope);
#pragma unroll
            for (int q = 0; q < V; ++q) v[q] = rs[q] * (g[q] * slope[q] * cp.gamma[q] - c1[q] - v[q] * c2[q]);
            store_acc<T, V>(dx + r * sh.channels + c, v);
        }
    }, [&](int64_t row, int64_t end) {
        const A zero[V] = {};
        for (int64_t r = row + row_lane; r < end; r += row_lanes) store_acc<T, V>(dx + r * sh.channels + c, zero);
    });
}
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) grad_apply_kernel(Shape sh, const T* __restrict__ x, const T* __restrict__ dy,
                                                              const T* __restrict__ w, const T* __restrict__ bias,
                                                              const acc_t<T>* __restrict__ mean, const acc_t<T>* __restrict__ rstd,
                                                              const acc_t<T>* __restrict__ coef, T* __restrict__ dx) {
    apply_grads<T, V, ACT>(sh, ChunkPieces{sh}, x, dy, w, bias, mean, rstd, coef, dx);
}

// The same for the segments that short_backward_kernel has handed over.  Without any, its lines of sums are zeros.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, 2) handed_backward_kernel(Shape sh, const T* __restrict__ x, const T* __restrict__ dy,
                                                                      const T* __restrict__ w, const T* __restrict__ bias,
                                                                      const acc_t<T>* __restrict__ mean, const acc_t<T>* __restrict__ rstd,
                                                                      acc_t<T>* part, acc_t<T>* block_sums, acc_t<T>* coef, T* __restrict__ dx) {
    __shared__ HandedPieces pieces;
    __shared__ double sm[kThreads / 32];
    pieces.find(sh);
    if (pieces.count == 0) {
        for (int c = threadIdx.x; blockIdx.y == 0 && c < 2 * sh.channels; c += kThreads) block_sums[blockIdx.x * int64_t(2) * sh.channels + c] = 0;
        return;
    }
    form_grad_sums<T, V, ACT>(sh, pieces, x, dy, w, bias, mean, rstd, part, block_sums);
    if (!dx) return;
    cooperative_groups::this_grid().sync();
    const int width = sh.channels / sh.groups, n = pieces.count * sh.groups;
    for (int item = blockIdx.y * gridDim.x + blockIdx.x; item < n; item += gridDim.x * gridDim.y) {
        const int q = item / sh.groups, g = item % sh.groups;
        const Span span{pieces.start[q], pieces.start[q + 1], pieces.chunk()};
        join_grads<T, kThreads>(span, true, part + (span.first() + q) * 2 * sh.channels + g * width, sh.channels, width,
                                w ? w + g * width : nullptr, sm, coef + 2 * (int64_t(pieces.segment[q]) * sh.groups + g));
    }
    cooperative_groups::this_grid().sync();
    apply_grads<T, V, ACT>(sh, pieces, x, dy, w, bias, mean, rstd, coef, dx);
}

// ---- short segments: one block per (segment, slab of whole groups), one launch per direction -------------------
// The rows of a short segment stay in L1 / L2 between the passes over them, so the block simply reads them again:
// once for the mean, once for the squared deviations from it, once to apply (backward: sums, then apply).

// Division of small numbers (n d < 2^32) by a number that the host knows.
struct Divisor {
    uint32_t d, magic;
    __host__ explicit Divisor(int v = 1) : d(v), magic(v > 1 ? 0xFFFFFFFFu / v + 1 : 0) {}
    __device__ __forceinline__ int div(int n) const { return d == 1 ? n : static_cast<int>(__umulhi(n, magic)); }
    __device__ __forceinline__ int mod(int n) const { return n - div(n) * static_cast<int>(d); }
};

struct Slab {
    int channels, lanes;          // channels of a slab (whole groups), vectors of its row
    int pad_blocks;               // blocks that write the rows outside every segment
    int64_t handed;               // see Shape
    int width, groups;            // channels of a group, groups of a slab
    Divisor by_lanes, by_width;
    // sums over a group: by one vector per column (width / V columns) in the forward pass, per channel in the backward
    int columns;
    Divisor by_parts, by_columns; // warps of a group; threads of a warp along a group's columns
    Divisor by_channels;
};

constexpr int kShort = 256;                         // threads of these blocks, and most channels of a slab
constexpr int kSlabGroups = kShort;                 // most groups of a slab

// Sum over the row lanes and over the columns of each group of sm [rows][groups * width].  The block's warps share the
// groups, several to a group when there are few; out holds `parts` sums per group.
template <typename A>
struct GroupSums {
    A out[kSlabGroups + kShort / 32];
    __device__ __forceinline__ void form(const A* sm, int rows, const Slab& slab, int width, const Divisor& by_columns) {
        const int p = slab.by_parts.d, lane = threadIdx.x % 32, line = slab.groups * width;
        const int per = by_columns.d, lanes = by_columns.div(32), row = by_columns.div(lane), column = lane - row * per;
        for (int item = threadIdx.x / 32; item < slab.groups * p; item += kShort / 32) {
            const int g = slab.by_parts.div(item), part = item - g * p;
            A v = 0;
            if (row < lanes)
                for (int r = part * lanes + row; r < rows; r += p * lanes)
                    for (int c = column; c < width; c += per) v += sm[r * line + g * width + c];
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
            if (lane == 0) out[item] = v;
        }
    }
    __device__ __forceinline__ A total(int g, const Slab& slab) const {
        const int p = slab.by_parts.d;
        A v = out[g * p];
        for (int q = 1; q < p; ++q) v += out[g * p + q];
        return v;
    }
};

template <typename T, int V>
__device__ __forceinline__ void zero_outside(const Shape& sh, int64_t first, int64_t blocks, T* out) {
    const acc_t<T> zero[V] = {};
    const int64_t before = segment_begin(sh, 0), behind = max(before, segment_begin(sh, sh.segments));
    const int64_t vectors = sh.channels / V, count = (before + sh.rows - behind) * vectors;
    for (int64_t e = first * kShort + threadIdx.x; e < count; e += blocks * kShort) {
        const int64_t r = e / vectors;
        store_acc<T, V>(out + (r < before ? r : r - before + behind) * sh.channels + e % vectors * V, zero);
    }
}

// What a block of the short segments has read of the row pointers, for the launch that takes the long ones: its blocks wait
// for one another at grid barriers, so they must not disagree about the segments, whatever happens to the row pointers
// meanwhile.
__device__ __forceinline__ void keep_pointers(const Shape& sh, int64_t* kept, int64_t s, int64_t begin) {
    if (kept == nullptr || blockIdx.y != 0 || threadIdx.x != 0) return;
    kept[s] = begin;
    if (s == sh.segments - 1) kept[sh.segments] = segment_begin(sh, sh.segments);
}

// ONE: a vector of channels belongs to one group (V divides channels / groups), so that a thread has one mean and one
// sum instead of V.
template <typename T, int V, int ACT, bool ONE>
__global__ void __launch_bounds__(kShort, 4) short_forward_kernel(Shape sh, Slab slab, const T* __restrict__ x, const T* __restrict__ w,
                                                               const T* __restrict__ bias, double eps, acc_t<T>* __restrict__ mean,
                                                               acc_t<T>* __restrict__ rstd, T* __restrict__ y, int64_t* __restrict__ kept) {
    using A = acc_t<T>;
    constexpr int G = ONE ? 1 : V;                                     // groups that a thread may touch
    __shared__ A sm[kShort * G], scale[kSlabGroups];
    __shared__ GroupSums<A> sums;
    if (blockIdx.x >= sh.segments) {
        if (blockIdx.y == 0) zero_outside<T, V>(sh, blockIdx.x - sh.segments, slab.pad_blocks, y);
        return;
    }
    const int64_t s = blockIdx.x, begin = segment_begin(sh, s), end = max(begin, segment_begin(sh, s + 1));
    const int width = slab.width, groups = slab.groups, first = blockIdx.y * slab.channels, g0 = blockIdx.y * groups;
    keep_pointers(sh, kept, s, begin);
    if (sh.handed != 0 && end - begin > sh.handed) return;
    if (end == begin) {
        for (int g = threadIdx.x; g < groups; g += kShort) mean[s * sh.groups + g0 + g] = rstd[s * sh.groups + g0 + g] = A(0);
        return;
    }
    const int row_lane = slab.by_lanes.div(threadIdx.x), lane = threadIdx.x - row_lane * slab.lanes, row_lanes = slab.by_lanes.div(kShort);
    const int c = lane * V;                                            // inside the slab
    const int used = static_cast<int>(min(int64_t(row_lanes), end - begin));       // row lanes that have a row
    const int64_t rows = row_lane < row_lanes ? end - begin : 0, step = int64_t(row_lanes) * sh.channels;
    const int64_t at = (begin + row_lane) * sh.channels + first + c;
    // columns of sm: one per vector (ONE) or per channel
    const int line = ONE ? slab.lanes : slab.channels;
    int group[G];
    A m[G], sum[G] = {};
#pragma unroll
    for (int q = 0; q < G; ++q) {
        group[q] = slab.by_width.div(c + q);
        m[q] = to_acc(x[begin * sh.channels + first + group[q] * width]);          // the group's first value
    }
    // several rows' loads under way at a time: the longest segment of a batch is bound by their latency
    auto over_rows = [&](auto&& f) {
        const T* p = x + at;
        int64_t r = row_lane;
        for (; r + 3 * int64_t(row_lanes) < rows; r += 4 * int64_t(row_lanes), p += 4 * step) {
            Pack<T, V> raw[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[e] = *reinterpret_cast<const Pack<T, V>*>(p + e * step);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                A v[V];
#pragma unroll
                for (int q = 0; q < V; ++q) v[q] = to_acc(raw[e].v[q]);
                f(v, p + e * step - x);
            }
        }
#pragma unroll 1
        for (; r < rows; r += row_lanes, p += step) {
            A v[V];
            load_acc<T, V>(p, v);
            f(v, p - x);
        }
    };
    auto join = [&]() {
        if (rows > 0)
#pragma unroll
            for (int q = 0; q < G; ++q) sm[row_lane * line + (ONE ? lane : c + q)] = sum[q];
        __syncthreads();
        sums.form(sm, used, slab, slab.columns, slab.by_columns);
        __syncthreads();
    };
    const A n = static_cast<A>(end - begin) * width;
    over_rows([&](const A (&v)[V], int64_t) {
#pragma unroll
        for (int q = 0; q < V; ++q) sum[ONE ? 0 : q] += v[q] - m[ONE ? 0 : q];
    });
    join();
#pragma unroll
    for (int q = 0; q < G; ++q) {
        m[q] += sums.total(group[q], slab) / n;
        sum[q] = 0;
        if (row_lane == 0 && group[q] * width == c + q) mean[s * sh.groups + g0 + group[q]] = m[q];
    }
    over_rows([&](const A (&v)[V], int64_t) {
#pragma unroll
        for (int q = 0; q < V; ++q) {
            const A d = v[q] - m[ONE ? 0 : q];
            sum[ONE ? 0 : q] += d * d;
        }
    });
    join();
    for (int g = threadIdx.x; g < groups; g += kShort) {
        scale[g] = static_cast<A>(1.0 / sqrt(static_cast<double>(sums.total(g, slab)) / static_cast<double>(n) + eps));
        rstd[s * sh.groups + g0 + g] = scale[g];
    }
    __syncthreads();
    A a[V], b[V];
    if (rows > 0)
#pragma unroll
        for (int q = 0; q < V; ++q) {
            a[q] = scale[group[ONE ? 0 : q]] * (w ? to_acc(w[first + c + q]) : A(1));
            b[q] = bias ? to_acc(bias[first + c + q]) : A(0);
        }
    over_rows([&](const A (&v)[V], int64_t offset) {
        A out[V];
#pragma unroll
        for (int q = 0; q < V; ++q) out[q] = (v[q] - m[ONE ? 0 : q]) * a[q] + b[q];
        activate_all<ACT>(out);
        store_acc<T, V>(y + offset, out);
    });
}

template <typename T, int V, int ACT, bool ONE>
__global__ void __launch_bounds__(kShort, sizeof(T) == 8 ? 2 : 4) short_backward_kernel(Shape sh, Slab slab, const T* __restrict__ x, const T* __restrict__ dy,
                                                                const T* __restrict__ w, const T* __restrict__ bias,
                                                                const acc_t<T>* __restrict__ mean, const acc_t<T>* __restrict__ rstd,
                                                                acc_t<T>* __restrict__ channel_sums, T* __restrict__ dx,
                                                                int64_t* __restrict__ kept) {
    using A = acc_t<T>;
    constexpr int G = ONE ? 1 : V;
    __shared__ A sm[kShort * V];
    __shared__ A weighted[2][kShort];
    __shared__ GroupSums<A> sums[2];
    if (blockIdx.x >= sh.segments) {
        if (dx && blockIdx.y == 0) zero_outside<T, V>(sh, blockIdx.x - sh.segments, slab.pad_blocks, dx);
        return;
    }
    const int64_t s = blockIdx.x, begin = segment_begin(sh, s), end = max(begin, segment_begin(sh, s + 1));
    const int width = slab.width, first = blockIdx.y * slab.channels, mine = slab.channels, g0 = blockIdx.y * slab.groups;
    keep_pointers(sh, kept, s, begin);
    if (sh.handed != 0 && end - begin > sh.handed) {     // its share of dbeta and dgamma is in another line
        if (threadIdx.x < mine)
            channel_sums[s * 2 * sh.channels + first + threadIdx.x] = channel_sums[s * 2 * sh.channels + sh.channels + first + threadIdx.x] = A(0);
        return;
    }
    const int row_lane = slab.by_lanes.div(threadIdx.x), lane = threadIdx.x - row_lane * slab.lanes, row_lanes = slab.by_lanes.div(kShort);
    const int c = lane * V;
    const int used = static_cast<int>(min(int64_t(row_lanes), end - begin));
    const int64_t rows = row_lane < row_lanes ? end - begin : 0, step = int64_t(row_lanes) * sh.channels;
    const int64_t at = (begin + row_lane) * sh.channels + first + c;
    A gamma[V], beta[V], m[G], rs[G];
    int group[G];
#pragma unroll
    for (int q = 0; q < V; ++q) {
        gamma[q] = w ? to_acc(w[first + c + q]) : A(1);
        beta[q] = bias ? to_acc(bias[first + c + q]) : A(0);
    }
#pragma unroll
    for (int q = 0; q < G; ++q) {
        group[q] = slab.by_width.div(c + q);
        m[q] = mean[s * sh.groups + g0 + group[q]];
        rs[q] = rstd[s * sh.groups + g0 + group[q]];
    }
    A s1[V] = {}, s2[V] = {};
    {
        const T *px = x + at, *pg = dy + at;
#pragma unroll 2
        for (int64_t r = row_lane; r < rows; r += row_lanes, px += step, pg += step) {
            A v[V], g[V];
            load_acc<T, V>(px, v);
            load_acc<T, V>(pg, g);
            A slope[V];
#pragma unroll
            for (int q = 0; q < V; ++q) {
                v[q] = (v[q] - m[ONE ? 0 : q]) * rs[ONE ? 0 : q];
                slope[q] = v[q] * gamma[q] + beta[q];
            }
            slope_all<ACT>(slope);
#pragma unroll
            for (int q = 0; q < V; ++q) {
                const A dz = g[q] * slope[q];
                s1[q] += dz;
                s2[q] += dz * v[q];
            }
        }
    }
    // sums over the row lanes: per channel for dbeta and dgamma, weighted with gamma per group for dx
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        if (row_lane < row_lanes)
#pragma unroll
            for (int q = 0; q < V; ++q) sm[row_lane * mine + c + q] = part == 0 ? s1[q] : s2[q];
        __syncthreads();
        if (threadIdx.x < mine) {
            const int ch = threadIdx.x;
            A v = 0;
#pragma unroll 8
            for (int r = 0; r < used; ++r) v += sm[r * mine + ch];
            channel_sums[s * 2 * sh.channels + part * sh.channels + first + ch] = v;
            weighted[part][ch] = v * (w ? to_acc(w[first + ch]) : A(1));
        }
        __syncthreads();
    }
    if (!dx) return;
    sums[0].form(weighted[0], 1, slab, width, slab.by_channels);
    sums[1].form(weighted[1], 1, slab, width, slab.by_channels);
    __syncthreads();
    A c1[G], c2[G];
    const A n = static_cast<A>(end - begin) * width;
#pragma unroll
    for (int q = 0; q < G; ++q) {
        c1[q] = sums[0].total(group[q], slab) / n;
        c2[q] = sums[1].total(group[q], slab) / n;
    }
    const T *px = x + at, *pg = dy + at;
    T* out = dx + at;
#pragma unroll 2
    for (int64_t r = row_lane; r < rows; r += row_lanes, px += step, pg += step, out += step) {
        A v[V], g[V];
        load_acc<T, V>(px, v);
        load_acc<T, V>(pg, g);
        A slope[V];
#pragma unroll
        for (int q = 0; q < V; ++q) {
            v[q] = (v[q] - m[ONE ? 0 : q]) * rs[ONE ? 0 : q];
            slope[q] = v[q] * gamma[q] + beta[q];
        }
        slope_all<ACT>(slope);
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = rs[ONE ? 0 : q] * (g[q] * slope[q] * gamma[q] - c1[ONE ? 0 : q] - v[q] * c2[ONE ? 0 : q]);
        store_acc<T, V>(out, v);
    }
}

// ---- host side ------------------------------------------------------------------------------------------
int64_t block_count(int64_t rows) {
    const int64_t wanted = ceil_div(rows, 32);
    return wanted < kSMs * 8 ? (wanted < 1 ? 1 : wanted) : kSMs * 8;
}

// Whether the one-block-per-segment kernels run, and with which slabs of channels.  They need segments that stay in
// a block's L1 on average (a slab of one up to 128 KB) and an array of at most 8 MB a slab; beyond that the row chunks
// take over.  A single block reads about 20 GB/s, so a long segment among short ones would be waited for: in an
// array above 512 KB a slab, segments above 128 KB a slab are handed over to one more launch,
// which finds none in most batches.  Measured, forward / backward of 61,441 rows x 128 bfloat16 in 512 graphs, one of
// which has all rows but 511: 47 / 76 us, with that graph in one block 581 / 1166, in row chunks 397 / 397; the launch
// costs equal graphs 4 us (23 -> 28 forward).  At 512 KB (8192 rows in 64 graphs) the long one in one block
// takes 48 / 92 us.
// Slabs are made narrower (whole groups) while there are fewer than eight blocks for
// every SM, down to rows of 64 bytes, or fewer than two, down to 32.  Measured on 512 graphs of 1 to 1076 rows, mean
// 118, x 128 bfloat16 channels with gelu, forward / backward: slabs of 128 channels 46 / 100 us, 64: 32 / 65, 32: 31 /
// 57, with four channels to a thread 31 / 51 (clusters of 2 to 8 blocks per graph were no faster: 34-41 / 67-72); the row
// chunks 82 / 117 us in six launches.  On other batches (2048 to 131,072 rows in 16 to 4096 graphs, equal and cut at random;
// 32 floats, 128 floats, 256 halves, 512 doubles) the row chunks take 1.0 to 5 times as long, but for 256 halves in graphs of
// 32 rows (0.7 forward, 1.04 backward) and 512 doubles at the limit (0.9).
constexpr int64_t kAlone = 512 * 1024, kInBlock = 128 * 1024;
bool short_segments(int64_t rows, int64_t channels, int64_t groups, int64_t segments, bool ragged, size_t size, int V, Slab* slab) {
    if (segments < 1 || segments > 65535 * 16) return false;
    const int64_t width = channels / groups;
    auto divisor = [&](int64_t most) {                                 // the largest divisor of groups up to it whose rows are whole vectors
        for (int64_t d = most; d >= 1; --d)
            if (groups % d == 0 && d * width % V == 0) return d;
        return int64_t(0);
    };
    const int64_t room = kShort / width;
    int64_t in_slab = divisor(groups < room ? groups : room);
    if (in_slab == 0) return false;
    for (;;) {
        const int64_t d = divisor(in_slab - 1), d_line = d * width * int64_t(size);
        const int64_t blocks = segments * (groups / in_slab);
        const bool few = (blocks < 8 * kSMs && d_line >= 64) || (blocks < 2 * kSMs && d_line >= 32);
        const bool heavy = rows * in_slab * width * int64_t(size) > 8 * 1024 * 1024 && d_line >= 64;
        if (d == 0 || !(few || heavy)) break;
        in_slab = d;
    }
    const int64_t line = in_slab * width * int64_t(size);
    if (rows / segments * line > kInBlock || rows * line > 8 * 1024 * 1024) return false;
    slab->handed = ragged && rows * line > kAlone ? kInBlock / line : 0;
    if (slab->handed != 0 && (ceil_div(rows, slab->handed) > kMostHanded || ceil_div(channels, kThreads) > 2 * kSMs)) return false;
    if (groups / in_slab > 65535) return false;
    slab->channels = static_cast<int>(in_slab * width);
    slab->lanes = static_cast<int>(in_slab * width / V);
    slab->width = static_cast<int>(width);
    slab->groups = static_cast<int>(in_slab);
    slab->by_lanes = Divisor(slab->lanes);
    slab->by_width = Divisor(slab->width);
    slab->columns = static_cast<int>(width % V == 0 ? width / V : width);
    slab->by_parts = Divisor(slab->groups < kShort / 32 ? kShort / 32 / slab->groups : 1);
    slab->by_columns = Divisor(slab->columns < 32 ? slab->columns : 32);
    slab->by_channels = Divisor(slab->width < 32 ? slab->width : 32);
    return true;
}

// The workspace: a line of 2 x channels values per block and per segment; one per block, and kMostHanded; two values per
// (segment, group); row pointers.  The first holds the pieces' partial results and the second the blocks' sums of dbeta and dgamma, or,
// in the backward pass over short segments, the first these sums per segment and per block, and the second the pieces.
size_t first_elements(int64_t rows, int64_t channels, int64_t segments) { return size_t(block_count(rows) + segments) * 2 * channels; }
size_t second_elements(int64_t rows, int64_t channels) { return size_t(block_count(rows) + kMostHanded) * 2 * channels; }
size_t elements(int64_t rows, int64_t channels, int64_t groups, int64_t segments) {
    return first_elements(rows, channels, segments) + second_elements(rows, channels) + size_t(segments) * groups * 2;
}
template <typename A>
int64_t* kept_pointers(int64_t rows, int64_t channels, int64_t groups, int64_t segments, A* work) {
    return reinterpret_cast<int64_t*>(work + elements(rows, channels, groups, segments));      // an even number of values: 8-byte aligned
}

bool bad_shape(int64_t rows, int64_t channels, int64_t groups, int64_t segments, const int64_t* ptr) {
    return rows < 0 || channels < 1 || channels > (1 << 20) || groups < 1 || channels % groups != 0 || segments < 0 ||
           segments > INT32_MAX || (!ptr && (segments < 1 ? rows != 0 : rows % segments != 0));
}

struct Launch {
    Shape sh;
    dim3 grid;
};

// Channels of a thread.  16-bit types: four, where a thread of eight would hold so much that too few are resident
// (a million rows of 128 bfloat16 forward 199 us against 234; the batch of short graphs backward 51 against 57), but
// eight in the backward pass over row chunks (392 us against 449).
template <typename T>
constexpr int few_channels() { return sizeof(T) == 2 ? 4 : 16 / sizeof(T); }

template <int V>
Launch make_launch(int64_t rows, int64_t channels, int64_t groups, int64_t segments, const int64_t* ptr) {
    Launch l;
    const int vectors = static_cast<int>(channels / V);
    const int64_t blocks = block_count(rows), chunk = ceil_div(rows, blocks);
    const int lanes = vectors < kThreads ? vectors : kThreads;
    l.sh = {rows, chunk, static_cast<int>(channels), static_cast<int>(groups), lanes, segments, ptr,
            segments > 0 ? rows / segments : rows, 0};
    l.grid = dim3(static_cast<unsigned>(ceil_div(rows, chunk)), static_cast<unsigned>(ceil_div(vectors, lanes)));
    return l;
}

template <typename T, int V>
int forward_chunks(const Launch& l, const T* x, const T* w, const T* b, double eps, int act, T* y, acc_t<T>* mean, acc_t<T>* rstd,
                   acc_t<T>* part, cudaStream_t stream) {
    using A = acc_t<T>;
    stats_kernel<T, V><<<l.grid, kThreads, 0, stream>>>(l.sh, x, part);
    const int64_t items = l.sh.segments * l.sh.groups;
    if (items > 0) {
        if (items > kSMs * 8)
            stats_join_kernel<A, 32><<<static_cast<unsigned>(ceil_div(items, kThreads / 32)), kThreads, 0, stream>>>(l.sh, part, eps, mean, rstd);
        else
            stats_join_kernel<A, 1024><<<static_cast<unsigned>(items), 1024, 0, stream>>>(l.sh, part, eps, mean, rstd);
    }
    return NB200_DISPATCH_ACT(act, (apply_kernel<T, V, ACT><<<l.grid, kThreads, 0, stream>>>(l.sh, x, w, b, mean, rstd, y),
                                    launch_status()));
}

// Blocks that are resident together, two to an SM; not more in a row than the row chunks' workspace is made for.
dim3 handed_grid(const Launch& l) {
    const unsigned row = 2 * kSMs / l.grid.y;
    return dim3(row < l.grid.x ? row : l.grid.x, l.grid.y);
}
template <typename... Params, typename... Args>
int launch_handed(void (*kernel)(Params...), dim3 grid, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeCooperative;
    attribute[0].val.cooperative = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...) == cudaSuccess ? launch_status() : NB200_ERR_CUDA;
}

template <typename T, int V>
int forward(Launch l, const T* x, const T* w, const T* b, double eps, int act, T* y, acc_t<T>* mean, acc_t<T>* rstd, acc_t<T>* part,
            cudaStream_t stream) {
    Slab slab;
    if (!short_segments(l.sh.rows, l.sh.channels, l.sh.groups, l.sh.segments, l.sh.ptr != nullptr, sizeof(T), V, &slab))
        return forward_chunks<T, V>(l, x, w, b, eps, act, y, mean, rstd, part, stream);
    slab.pad_blocks = l.sh.ptr ? kSMs / 4 : 0;
    l.sh.handed = slab.handed;
    int64_t* kept = slab.handed != 0 ? kept_pointers(l.sh.rows, l.sh.channels, l.sh.groups, l.sh.segments, part) : nullptr;
    const dim3 grid(static_cast<unsigned>(l.sh.segments + slab.pad_blocks), static_cast<unsigned>(l.sh.channels / slab.channels));
    const int rc = l.sh.channels / l.sh.groups % V == 0
                       ? NB200_DISPATCH_ACT(act, (short_forward_kernel<T, V, ACT, true><<<grid, kShort, 0, stream>>>(l.sh, slab, x, w, b, eps, mean,
                                                                                                                   rstd, y, kept), launch_status()))
                       : NB200_DISPATCH_ACT(act, (short_forward_kernel<T, V, ACT, false><<<grid, kShort, 0, stream>>>(l.sh, slab, x, w, b, eps, mean,
                                                                                                                    rstd, y, kept), launch_status()));
    if (rc != NB200_OK || slab.handed == 0) return rc;
    l.sh.ptr = kept;
    return NB200_DISPATCH_ACT(act, launch_handed(handed_forward_kernel<T, V, ACT>, handed_grid(l), stream, l.sh, x, w, b, eps, mean, rstd, part, y));
}

template <typename T, int V>
int backward_short(const Launch& l, Slab slab, const T* dy, const T* x, const T* w, const T* b, const acc_t<T>* mean, const acc_t<T>* rstd,
                   int act, T* dx, acc_t<T>* segment_sums, int64_t* kept, cudaStream_t stream) {
    slab.pad_blocks = l.sh.ptr && dx ? kSMs / 4 : 0;
    const dim3 grid(static_cast<unsigned>(l.sh.segments + slab.pad_blocks), static_cast<unsigned>(l.sh.channels / slab.channels));
    return l.sh.channels / l.sh.groups % V == 0
               ? NB200_DISPATCH_ACT(act, (short_backward_kernel<T, V, ACT, true><<<grid, kShort, 0, stream>>>(
                                              l.sh, slab, x, dy, w, b, mean, rstd, segment_sums, dx, kept), launch_status()))
               : NB200_DISPATCH_ACT(act, (short_backward_kernel<T, V, ACT, false><<<grid, kShort, 0, stream>>>(
                                              l.sh, slab, x, dy, w, b, mean, rstd, segment_sums, dx, kept), launch_status()));
}

// Up to dx; dbeta and dgamma are left as one line of sums per block.
template <typename T, int V>
int backward_chunks(const Launch& l, const T* dy, const T* x, const T* w, const T* b, const acc_t<T>* mean, const acc_t<T>* rstd, int act,
                    T* dx, acc_t<T>* part, acc_t<T>* block_sums, acc_t<T>* coef, cudaStream_t stream) {
    const int rc = NB200_DISPATCH_ACT(act, (grad_sums_kernel<T, V, ACT><<<l.grid, kThreads, 0, stream>>>(
                                                l.sh, x, dy, w, b, mean, rstd, part, block_sums), launch_status()));
    if (rc != NB200_OK || !dx) return rc;
    const int64_t items = l.sh.segments * l.sh.groups;
    if (items > 0) {
        if (items > kSMs * 8)
            grad_join_kernel<T, 32><<<static_cast<unsigned>(ceil_div(items, kThreads / 32)), kThreads, 0, stream>>>(l.sh, part, w, coef);
        else
            grad_join_kernel<T, 1024><<<static_cast<unsigned>(items), 1024, 0, stream>>>(l.sh, part, w, coef);
    }
    return NB200_DISPATCH_ACT(act, (grad_apply_kernel<T, V, ACT><<<l.grid, kThreads, 0, stream>>>(l.sh, x, dy, w, b, mean, rstd, coef,
                                                                                                        dx), launch_status()));
}

// W: channels of a thread in the row chunks, V: in the blocks of short segments.
template <typename T, int V, int W>
int backward(int64_t rows, int64_t channels, int64_t groups, int64_t segments, const int64_t* ptr, const T* dy, const T* x, const T* w,
             const T* b, const acc_t<T>* mean, const acc_t<T>* rstd, int act, T* dx, T* dw, T* db, acc_t<T>* at, cudaStream_t stream) {
    acc_t<T>*first = at, *second = first + first_elements(rows, channels, segments), *coef = second + second_elements(rows, channels);
    Launch chunks = make_launch<W>(rows, channels, groups, segments, ptr);
    Slab slab;
    const acc_t<T>* lines;
    int64_t count;
    int rc;
    if (short_segments(rows, channels, groups, segments, ptr != nullptr, sizeof(T), V, &slab)) {
        Launch blocks = make_launch<V>(rows, channels, groups, segments, ptr);
        blocks.sh.handed = chunks.sh.handed = slab.handed;
        int64_t* kept = slab.handed != 0 ? kept_pointers(rows, channels, groups, segments, at) : nullptr;
        rc = backward_short<T, V>(blocks, slab, dy, x, w, b, mean, rstd, act, dx, first, kept, stream);
        lines = first;
        count = segments;
        if (rc == NB200_OK && slab.handed != 0) {
            const dim3 grid = handed_grid(chunks);
            chunks.sh.ptr = kept;
            rc = NB200_DISPATCH_ACT(act, launch_handed(handed_backward_kernel<T, W, ACT>, grid, stream, chunks.sh, x, dy, w, b, mean, rstd, second,
                                                       first + size_t(segments) * 2 * channels, coef, dx));
            count += grid.x;
        }
    } else {
        rc = backward_chunks<T, W>(chunks, dy, x, w, b, mean, rstd, act, dx, first, second, coef, stream);
        lines = second;
        count = chunks.grid.x;
    }
    if (rc != NB200_OK || !(dw || db)) return rc;
    column_sums_kernel<T><<<static_cast<unsigned>(ceil_div(2 * channels, 32)), 1024, 0, stream>>>(count, static_cast<int>(channels), lines, db, dw);
    return launch_status();
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" size_t nb200_group_norm_workspace_bytes(int64_t rows, int64_t channels, int64_t groups, int64_t segments, int dtype) {
    if (rows < 0 || channels < 1 || groups < 1 || segments < 0) return 0;
    const size_t a = dtype == NB200_F64 ? 8 : 4;
    return a * elements(rows, channels, groups, segments) + sizeof(int64_t) * (size_t(segments) + 1);
}

extern "C" int nb200_group_norm_forward(int64_t rows, int64_t channels, int64_t groups, int64_t segments, const int64_t* ptr,
                                        const void* x, const void* weight, const void* bias, double eps, int activation, void* y,
                                        void* mean, void* rstd, void* work, size_t work_bytes, int dtype, nb200_stream stream) {
    if (bad_shape(rows, channels, groups, segments, ptr) || !known_dense_dtype(dtype) || !known_activation(activation) || !(eps >= 0.0))
        return NB200_ERR_BAD_ARG;
    if (rows == 0 && segments == 0) return NB200_OK;
    if ((segments > 0 && (!mean || !rstd)) || !work || (rows > 0 && (!x || !y))) return NB200_ERR_BAD_ARG;
    if (work_bytes < nb200_group_norm_workspace_bytes(rows, channels, groups, segments, dtype)) return NB200_ERR_WORKSPACE;
    if (!aligned16(x) || !aligned16(y) || !aligned16(work)) return NB200_ERR_ALIGN;
    if (rows == 0) {
        const size_t bytes = size_t(segments) * groups * (dtype == NB200_F64 ? 8 : 4);
        if (cudaMemsetAsync(mean, 0, bytes, as_stream(stream)) != cudaSuccess ||
            cudaMemsetAsync(rstd, 0, bytes, as_stream(stream)) != cudaSuccess)
            return NB200_ERR_CUDA;
        return NB200_OK;
    }
    return NB200_DISPATCH_DENSE(dtype, ([&]() -> int {
        using A = acc_t<T>;
        const T *xt = static_cast<const T*>(x), *wt = static_cast<const T*>(weight), *bt = static_cast<const T*>(bias);
        A *m = static_cast<A*>(mean), *rs = static_cast<A*>(rstd), *part = static_cast<A*>(work);
        T* yt = static_cast<T*>(y);
        constexpr int V = few_channels<T>();
        return channels % V == 0 ? forward<T, V>(make_launch<V>(rows, channels, groups, segments, ptr), xt, wt, bt, eps, activation, yt, m, rs,
                                                 part, as_stream(stream))
                                 : forward<T, 1>(make_launch<1>(rows, channels, groups, segments, ptr), xt, wt, bt, eps, activation, yt, m, rs,
                                                 part, as_stream(stream));
    }()));
}

extern "C" int nb200_group_norm_backward(int64_t rows, int64_t channels, int64_t groups, int64_t segments, const int64_t* ptr,
                                         const void* dy, const void* x, const void* weight, const void* bias, const void* mean,
                                         const void* rstd, int activation, void* dx, void* dweight, void* dbias, void* work,
                                         size_t work_bytes, int dtype, nb200_stream stream) {
    if (bad_shape(rows, channels, groups, segments, ptr) || !known_dense_dtype(dtype) || !known_activation(activation))
        return NB200_ERR_BAD_ARG;
    if (rows == 0) {
        const size_t bytes = size_t(channels) * dense_dtype_size(dtype);
        if ((dweight && cudaMemsetAsync(dweight, 0, bytes, as_stream(stream)) != cudaSuccess) ||
            (dbias && cudaMemsetAsync(dbias, 0, bytes, as_stream(stream)) != cudaSuccess))
            return NB200_ERR_CUDA;
        return NB200_OK;
    }
    if (!x || !dy || (segments > 0 && (!mean || !rstd)) || !work) return NB200_ERR_BAD_ARG;
    if (work_bytes < nb200_group_norm_workspace_bytes(rows, channels, groups, segments, dtype)) return NB200_ERR_WORKSPACE;
    if (!aligned16(x) || !aligned16(dy) || !aligned16(work) || (dx && !aligned16(dx))) return NB200_ERR_ALIGN;
    return NB200_DISPATCH_DENSE(dtype, ([&]() -> int {
        using A = acc_t<T>;
        const T *xt = static_cast<const T*>(x), *gt = static_cast<const T*>(dy), *wt = static_cast<const T*>(weight),
                *bt = static_cast<const T*>(bias);
        const A *m = static_cast<const A*>(mean), *rs = static_cast<const A*>(rstd);
        A* part = static_cast<A*>(work);
        T *dxt = static_cast<T*>(dx), *dwt = static_cast<T*>(dweight), *dbt = static_cast<T*>(dbias);
        constexpr int V = few_channels<T>(), W = 16 / sizeof(T);
        auto run = [&](auto v, auto u) {
            return backward<T, decltype(v)::value, decltype(u)::value>(rows, channels, groups, segments, ptr, gt, xt, wt, bt, m, rs, activation, dxt,
                                                                       dwt, dbt, part, as_stream(stream));
        };
        using One = std::integral_constant<int, 1>;
        if (channels % W == 0) return run(std::integral_constant<int, V>(), std::integral_constant<int, W>());
        if (channels % V == 0) return run(std::integral_constant<int, V>(), One());
        return run(One(), One());
    }()));
}
