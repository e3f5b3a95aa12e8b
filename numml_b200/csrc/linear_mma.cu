// Dense products on the 5th-generation tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// float: the tensor cores multiply 8-bit significands (bfloat16) exactly and add in 32 bits, so a float is
// split into three bfloat16 pieces of 8 bits each, x = x0 + x1 + x2 (each piece the rounding of what the
// ones before leave, exact to 24 bits), and a product takes the six pairs of pieces whose weight is not
// below the last bit: x0y0, x0y1, x1y0, x1y1, x0y2, x2y0.  What is dropped is below 2^-25 of |x||y| per
// term, under the rounding of one float multiply-add.  bfloat16 and half go in as they are.
//
// One persistent block per SM, warps specialised: eight loader warps bring chunks of 64 terms of both
// operands into shared memory (float: through registers, split on the way; 16-bit types: asynchronous
// copies), one thread issues the products, eight epilogue warps take finished accumulators out of tensor
// memory, turn them so that a row is written in whole 128-byte lines, and apply bias, activation, residual
// and rounding.  Accumulators are double-buffered, so the products of a tile run under the epilogue of the
// one before.  When a tile's second operand fits beside the ring of the first (the weights of a layer with
// few channels), it is loaded and split once per block and the rows stream past it.
//
// The tensor cores truncate where they add, always towards zero.  For float the products of leading pieces
// therefore have an accumulator of their own, into which one addition goes per 16 terms (the five smaller ones
// go to a second, where a truncation weighs 2^-8 as much), and both are taken out every kDrainChunks chunks
// and added up in registers with rounding to nearest.
#include <type_traits>

#include "linear_mma.cuh"
#include "tcgen05.cuh"

namespace nb200 {
namespace {

constexpr int kEpilogueWarps = 8, kLoaderWarps = 8, kLoaders = kLoaderWarps * 32;
constexpr int kThreads = (kEpilogueWarps + kLoaderWarps + 1) * 32;
constexpr int kPieceBytes = kMmaTile * kMmaChunk * 2;              // one piece of one operand's chunk: 16 KB
constexpr int kUnits = kMmaTile * kMmaChunk / 8 / kLoaders;        // units of eight values per loader thread
constexpr int kDrainChunks = 2;

template <typename T> struct Traits {                              // 16-bit types
    static constexpr int pieces = 1, a_slots = 4, b_slots = 8, accumulators = 1;
    static constexpr bool drains = false;
};
template <> struct Traits<float> {
    static constexpr int pieces = 3, a_slots = 2, b_slots = 2, accumulators = 2;
    static constexpr bool drains = true;
};

template <typename T>
constexpr uint32_t tmem_columns() { return 2 * Traits<T>::accumulators * kMmaTile; }      // two buffers of each
template <typename T>
constexpr int slot_bytes() { return Traits<T>::pieces * kPieceBytes; }
template <typename T>
constexpr int smem_bytes() {
    return 1024 + (Traits<T>::a_slots + Traits<T>::b_slots) * slot_bytes<T>() + kEpilogueWarps * 4096;
}

struct Control {
    uint64_t full[8], empty[8], acc_full[2], acc_empty[2], done;
    uint32_t tmem;
    int gave_up;
};

template <typename T>
struct Operand {
    const T* p;
    int64_t ld, extent;       // row stride; rows (A) or columns (B) in all
    bool vector;              // base and stride are multiples of 16 bytes
};

template <typename T>
struct Args {
    Operand<T> a, b;
    int64_t rows, cols, depth, per;
    int64_t row_tiles, col_tiles, items;
    int chunks;               // chunks of the longest part of the sum
    bool resident, vector_out;
    Epilogue<T> ep;
    int32_t* status;
};

// ---- one unit of eight consecutive values (along k or along mn) ----------------------------------------
template <typename T, bool K_MAJOR>
struct UnitPlace {
    // position of unit q of this thread inside a 128 x 64 chunk
    static __device__ __forceinline__ int mn(int t, int q) { return K_MAJOR ? t / 8 + q * (kLoaders / 8) : (t % 16) * 8; }
    static __device__ __forceinline__ int k(int t, int q) { return K_MAJOR ? (t % 8) * 8 : t / 16 + q * (kLoaders / 16); }
    static __device__ __forceinline__ uint32_t offset(int t, int q) {
        const int m = mn(t, q), kk = k(t, q);
        if (K_MAJOR) return (m / 8) * 1024 + (m % 8) * 128 + (((kk / 8) ^ (m % 8)) * 16);
        return (m / 64) * (kPieceBytes / 2) + (kk / 8) * 1024 + (kk % 8) * 128 + ((((m % 64) / 8) ^ (kk % 8)) * 16);
    }
    // how many of the unit's values exist, given the ends of both ranges
    static __device__ __forceinline__ int valid(int64_t m, int64_t k, int64_t extent, int64_t k_end) {
        const int64_t line = K_MAJOR ? extent - m : k_end - k, run = K_MAJOR ? k_end - k : extent - m;
        return line <= 0 || run <= 0 ? 0 : (run < 8 ? static_cast<int>(run) : 8);
    }
    static __device__ __forceinline__ const T* address(const Operand<T>& o, int64_t m, int64_t k) {
        return K_MAJOR ? o.p + m * o.ld + k : o.p + k * o.ld + m;
    }
};

template <bool K_MAJOR>
__device__ __forceinline__ void fetch(const Operand<float>& o, int64_t m, int64_t k, int64_t k_end, float (&v)[8]) {
    using U = UnitPlace<float, K_MAJOR>;
    const int valid = U::valid(m, k, o.extent, k_end);
    const float* p = U::address(o, m, k);
    if (valid == 8 && o.vector) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = q < valid ? __ldg(p + q) : 0.f;
    }
}

// Eight floats as three pieces of eight bfloat16.
__device__ __forceinline__ void split_store(uint32_t addr, const float (&v)[8]) {
    uint32_t piece[3][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float lo = v[2 * q], hi = v[2 * q + 1];
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
            const uint32_t bits = *reinterpret_cast<const uint32_t*>(&r);
            piece[s][q] = bits;
            lo -= __uint_as_float(bits << 16);
            hi -= __uint_as_float(bits & 0xFFFF0000u);
        }
    }
#pragma unroll
    for (int s = 0; s < 3; ++s)
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(addr + s * kPieceBytes), "r"(piece[s][0]), "r"(piece[s][1]),
                     "r"(piece[s][2]), "r"(piece[s][3]) : "memory");
}

template <typename T, bool K_MAJOR>
__device__ __forceinline__ void copy_units(const Operand<T>& o, uint32_t slot, int t, int64_t m0, int64_t k0, int64_t k_end) {
    using U = UnitPlace<T, K_MAJOR>;
#pragma unroll
    for (int q = 0; q < kUnits; ++q) {
        const int64_t m = m0 + U::mn(t, q), k = k0 + U::k(t, q);
        const int valid = U::valid(m, k, o.extent, k_end);
        const T* p = valid > 0 ? U::address(o, m, k) : o.p;
        const uint32_t dst = slot + U::offset(t, q);
        if (o.vector) {
            tc::copy16(dst, p, valid * 2);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t lo = 2 * e < valid ? __ldg(reinterpret_cast<const unsigned short*>(p) + 2 * e) : 0u;
                const uint32_t hi = 2 * e + 1 < valid ? __ldg(reinterpret_cast<const unsigned short*>(p) + 2 * e + 1) : 0u;
                w[e] = lo | hi << 16;
            }
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        }
    }
}

// Walks the (item, chunk) sequence of a block; every role steps through it alike.
template <typename T>
struct Walk {
    const Args<T>& g;
    int64_t item;
    int64_t i0, j0, k_begin, k_end, split;
    int chunks, chunk;
    __device__ __forceinline__ explicit Walk(const Args<T>& args) : g(args), item(blockIdx.x), chunk(0) { place(); }
    __device__ __forceinline__ bool live() const { return item < g.items; }
    __device__ __forceinline__ void place() {
        if (!live()) return;
        const int64_t tile = item % (g.row_tiles * g.col_tiles);
        split = item / (g.row_tiles * g.col_tiles);
        j0 = tile % g.col_tiles * kMmaTile;
        i0 = tile / g.col_tiles * kMmaTile;
        k_begin = split * g.per;
        k_end = min(g.depth, k_begin + g.per);
        chunks = static_cast<int>((k_end - k_begin + kMmaChunk - 1) / kMmaChunk);
        if (chunks < 1) chunks = 1;                     // an empty sum is a chunk of zeros
    }
    __device__ __forceinline__ void next_item() {
        item += gridDim.x;
        chunk = 0;
        place();
    }
    __device__ __forceinline__ void next_chunk() {
        if (++chunk == chunks) next_item();
    }
};

template <typename T, bool A_K, bool B_K>
__device__ void load_role(const Args<T>& g, uint32_t a_ring, uint32_t b_ring, Control* ctl) {
    using Tr = Traits<T>;
    constexpr int S = Tr::a_slots;
    const int t = threadIdx.x - kEpilogueWarps * 32;
    Walk<T> w(g);
    bool first = true;                                   // the block's first item loads the resident operand
    if constexpr (Tr::pieces == 3) {
        // registers hold the units of the next chunk; a unit is refilled right after it has been stored
        float ra[kUnits][8], rb[kUnits][8];
        Walk<T> ahead(g);
        bool ahead_b = true;
        auto fetch_a = [&](int q) {
            fetch<A_K>(g.a, ahead.i0 + UnitPlace<T, A_K>::mn(t, q),
                       ahead.k_begin + ahead.chunk * kMmaChunk + UnitPlace<T, A_K>::k(t, q), ahead.k_end, ra[q]);
        };
        auto fetch_b = [&](int q) {
            fetch<B_K>(g.b, ahead.j0 + UnitPlace<T, B_K>::mn(t, q),
                       ahead.k_begin + ahead.chunk * kMmaChunk + UnitPlace<T, B_K>::k(t, q), ahead.k_end, rb[q]);
        };
        if (ahead.live()) {
#pragma unroll
            for (int q = 0; q < kUnits; ++q) {
                fetch_a(q);
                fetch_b(q);
            }
        }
        for (int64_t step = 0; w.live(); ++step) {
            const int slot = static_cast<int>(step % S);
            if (step >= S && !tc::mbar_wait(&ctl->empty[slot], static_cast<unsigned>((step / S - 1) & 1), &ctl->gave_up)) return;
            const int64_t item_now = ahead.item;
            ahead.next_chunk();
            if (ahead.item != item_now && g.resident) ahead_b = false;
            const bool with_b = !g.resident || first;
            const uint32_t b_slot = b_ring + (g.resident ? w.chunk : slot) * slot_bytes<T>();
#pragma unroll
            for (int q = 0; q < kUnits; ++q) {
                split_store(a_ring + slot * slot_bytes<T>() + UnitPlace<T, A_K>::offset(t, q), ra[q]);
                if (ahead.live()) fetch_a(q);
            }
            if (with_b) {
#pragma unroll
                for (int q = 0; q < kUnits; ++q) {
                    split_store(b_slot + UnitPlace<T, B_K>::offset(t, q), rb[q]);
                    if (ahead.live() && ahead_b) fetch_b(q);
                }
            }
            tc::fence_smem_for_async();
            __syncwarp();
            if (threadIdx.x % 32 == 0) tc::mbar_arrive(&ctl->full[slot]);
            const int64_t item = w.item;
            w.next_chunk();
            if (w.item != item) first = false;
        }
    } else {
        // copies of chunk n are announced S - 1 chunks later, when they have landed
        constexpr int LAG = S - 1;
        int64_t step = 0;
        bool ok = true;
        for (; w.live(); ++step) {
            const int slot = static_cast<int>(step % S);
            if (step >= S && !tc::mbar_wait(&ctl->empty[slot], static_cast<unsigned>((step / S - 1) & 1), &ctl->gave_up)) {
                ok = false;
                break;
            }
            const int64_t k0 = w.k_begin + w.chunk * kMmaChunk;
            copy_units<T, A_K>(g.a, a_ring + slot * slot_bytes<T>(), t, w.i0, k0, w.k_end);
            if (!g.resident || first)
                copy_units<T, B_K>(g.b, b_ring + (g.resident ? w.chunk : slot) * slot_bytes<T>(), t, w.j0, k0, w.k_end);
            tc::copy_commit();
            if (step >= LAG) {
                tc::copy_wait<LAG>();
                tc::fence_smem_for_async();
                __syncwarp();
                if (threadIdx.x % 32 == 0) tc::mbar_arrive(&ctl->full[(step - LAG) % S]);
            }
            const int64_t item = w.item;
            w.next_chunk();
            if (w.item != item) first = false;
        }
        tc::copy_wait<0>();
        tc::fence_smem_for_async();
        __syncwarp();
        if (ok && threadIdx.x % 32 == 0)
            for (int64_t s = step > LAG ? step - LAG : 0; s < step; ++s) tc::mbar_arrive(&ctl->full[s % S]);
    }
}

template <typename T, bool A_K, bool B_K>
__device__ void product_role(const Args<T>& g, uint32_t a_ring, uint32_t b_ring, uint32_t tmem, Control* ctl) {
    using Tr = Traits<T>;
    constexpr int S = Tr::a_slots;
    constexpr uint32_t idesc = tc::instruction_descriptor(!std::is_same<T, __half>::value, !A_K, !B_K, kMmaTile);
    constexpr uint32_t a_step = A_K ? 32 : 2048, b_step = B_K ? 32 : 2048;       // bytes from one 16-term step to the next
    int64_t groups = 0;                                                         // accumulators handed over so far
    int64_t step = 0;
    bool ok = true;
    for (Walk<T> w(g); ok && w.live(); w.next_item()) {
        for (int c = 0; ok && c < w.chunks; ++c, ++step) {
            const int slot = static_cast<int>(step % S), buffer = static_cast<int>(groups & 1);
            const bool fresh = Tr::drains ? c % kDrainChunks == 0 : c == 0;
            const bool last = c + 1 == w.chunks || (Tr::drains && (c + 1) % kDrainChunks == 0);
            if (fresh && groups >= 2) ok = tc::mbar_wait(&ctl->acc_empty[buffer], static_cast<unsigned>((groups / 2 - 1) & 1), &ctl->gave_up);
            ok = ok && tc::mbar_wait(&ctl->full[slot], static_cast<unsigned>((step / S) & 1), &ctl->gave_up);
            if (!ok) break;
            tc::fence_after_sync();
            const uint32_t a = a_ring + slot * slot_bytes<T>(), b = b_ring + (g.resident ? c : slot) * slot_bytes<T>();
            const uint32_t d = tmem + buffer * Tr::accumulators * kMmaTile;
            bool accumulate[2] = {!fresh, !fresh};
#pragma unroll
            for (int k = 0; k < kMmaChunk / 16; ++k) {
                auto product = [&](int pa, int pb) {
                    const uint64_t da = A_K ? tc::smem_descriptor(a + pa * kPieceBytes + k * a_step, 16, 1024)
                                            : tc::smem_descriptor(a + pa * kPieceBytes + k * a_step, kPieceBytes / 2, 1024);
                    const uint64_t db = B_K ? tc::smem_descriptor(b + pb * kPieceBytes + k * b_step, 16, 1024)
                                            : tc::smem_descriptor(b + pb * kPieceBytes + k * b_step, kPieceBytes / 2, 1024);
                    const int into = pa + pb > 0 ? 1 : 0;
                    tc::mma_f16(d + into * kMmaTile, da, db, idesc, accumulate[into]);
                    accumulate[into] = true;
                };
                if (Tr::pieces == 3) {
                    product(2, 0);
                    product(0, 2);
                    product(1, 1);
                    product(1, 0);
                    product(0, 1);
                }
                product(0, 0);
            }
            tc::commit(&ctl->empty[slot]);
            if (last) {
                tc::commit(&ctl->acc_full[buffer]);
                ++groups;
            }
        }
    }
    // nothing of this thread's may be in flight when tensor memory is given back
    tc::commit(&ctl->done);
    const uint32_t addr = tc::smem_u32(&ctl->done);
    const long long t0 = clock64();
    while (!tc::mbar_try(addr, 0) && clock64() - t0 < tc::kWaitCycles) {}
}

// An element in plain 32-bit arithmetic: taken when the pieces of an infinity, or of a value that rounds to
// one in 16 bits, have made a NaN of it.
template <typename T, bool A_K, bool B_K>
__device__ __noinline__ float plain_element(const Args<T>& g, int64_t i, int64_t j, int64_t k_begin, int64_t k_end) {
    float v = 0.f;
    for (int64_t k = k_begin; k < k_end; ++k)
        v = fmaf(to_acc(A_K ? g.a.p[i * g.a.ld + k] : g.a.p[k * g.a.ld + i]), to_acc(B_K ? g.b.p[j * g.b.ld + k] : g.b.p[k * g.b.ld + j]), v);
    return v;
}

template <typename T, bool A_K, bool B_K, int ACT>
__device__ __forceinline__ void write_rows(const Args<T>& g, const Walk<T>& w, uint32_t stage, int64_t row0, int64_t col0) {
    const int lane = threadIdx.x % 32;
    const int64_t j = col0 + (lane % 8) * 4;
    const Epilogue<T>& ep = g.ep;
    if (j >= g.cols) return;
    const int width = g.cols - j < 4 ? static_cast<int>(g.cols - j) : 4;
    float bias[4] = {};
    if (ep.bias)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < width) bias[q] = to_acc(ep.bias[j + q]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int r = lane / 8 + 4 * e;
        const int64_t i = row0 + r;
        if (i >= g.rows) break;
        float v[4];
        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                     : "r"(stage + r * 128 + (((lane % 8) ^ (r % 8)) * 16)));
        if (Traits<T>::pieces == 3) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (!isfinite(v[q]) && q < width) v[q] = plain_element<T, A_K, B_K>(g, i, j + q, w.k_begin, w.k_end);
        }
        if (ep.partial) {
            float* out = reinterpret_cast<float*>(ep.partial) + (w.split * g.rows + i) * g.cols + j;
            if (g.vector_out) {
                *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (q < width) out[q] = v[q];
            }
            continue;
        }
        float res[4] = {};
        if (ep.residual) {
            const T* p = ep.residual + i * ep.ldr + j;
            if (g.vector_out) {
                load_acc<T, 4>(p, res);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (q < width) res[q] = to_acc(p[q]);
            }
        }
        Pack<T, 4> z, y;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float s = v[q] + bias[q];
            z.v[q] = rounded_z<T, ACT>(s);
            float t = activate<ACT>(s);
            if (ep.residual) t += res[q];
            y.v[q] = from_acc<T>(t);
        }
        if (g.vector_out) {
            if (ep.z) *reinterpret_cast<Pack<T, 4>*>(ep.z + i * g.cols + j) = z;
            *reinterpret_cast<Pack<T, 4>*>(ep.y + i * g.cols + j) = y;
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q < width) {
                    if (ep.z) ep.z[i * g.cols + j + q] = z.v[q];
                    ep.y[i * g.cols + j + q] = y.v[q];
                }
        }
    }
}

template <typename T, bool A_K, bool B_K, int ACT>
__device__ void epilogue_role(const Args<T>& g, uint32_t staging, uint32_t tmem, Control* ctl) {
    using Tr = Traits<T>;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int quarter = warp % 4, half = warp / 4;                 // tensor memory lanes and columns of this warp
    const uint32_t stage = staging + warp * 4096;
    int64_t groups = 0;
    for (Walk<T> w(g); w.live(); w.next_item()) {
        float acc[Tr::drains ? 64 : 1];
        const int parts = Tr::drains ? (w.chunks + kDrainChunks - 1) / kDrainChunks : 1;
        for (int part = 0; part < parts; ++part, ++groups) {
            const int buffer = static_cast<int>(groups & 1);
            if (!tc::mbar_wait(&ctl->acc_full[buffer], static_cast<unsigned>((groups / 2) & 1), &ctl->gave_up)) return;
            tc::fence_after_sync();
#pragma unroll
            for (int block = 0; block < 2; ++block) {
                float v[32];
                const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + buffer * Tr::accumulators * kMmaTile + half * 64 + block * 32;
                tc::tmem_load32(from, v);
                if constexpr (Tr::drains) {
                    float small[32];
                    tc::tmem_load32(from + kMmaTile, small);
#pragma unroll
                    for (int q = 0; q < 32; ++q) v[q] += small[q];
#pragma unroll
                    for (int q = 0; q < 32; ++q) acc[block * 32 + q] = part == 0 ? v[q] : acc[block * 32 + q] + v[q];
                    if (part + 1 < parts) continue;
#pragma unroll
                    for (int q = 0; q < 32; ++q) v[q] = acc[block * 32 + q];
                }
                __syncwarp();                                        // the block before has been read out of the stage
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" :: "r"(stage + lane * 128 + ((q ^ (lane % 8)) * 16)), "f"(v[4 * q]),
                                 "f"(v[4 * q + 1]), "f"(v[4 * q + 2]), "f"(v[4 * q + 3]) : "memory");
                __syncwarp();
                if (block == 1) {                                    // everything has left tensor memory
                    tc::fence_before_sync();
                    if (lane == 0) tc::mbar_arrive(&ctl->acc_empty[buffer]);
                }
                write_rows<T, A_K, B_K, ACT>(g, w, stage, w.i0 + quarter * 32, w.j0 + half * 64 + block * 32);
            }
            if (Tr::drains && part + 1 < parts) {
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&ctl->acc_empty[buffer]);
            }
        }
    }
}

template <typename T, bool A_K, bool B_K, int ACT>
__global__ void __launch_bounds__(kThreads, 1) mma_kernel(const __grid_constant__ Args<T> g) {
    using Tr = Traits<T>;
    extern __shared__ char raw[];
    __shared__ Control ctl;
    const uint32_t base = (tc::smem_u32(raw) + 1023) / 1024 * 1024;
    const uint32_t a_ring = base, b_ring = a_ring + Tr::a_slots * slot_bytes<T>(), staging = b_ring + Tr::b_slots * slot_bytes<T>();
    const int warp = threadIdx.x / 32;
    if (threadIdx.x == 0) {
        for (int s = 0; s < Tr::a_slots; ++s) {
            tc::mbar_init(&ctl.full[s], kLoaderWarps);
            tc::mbar_init(&ctl.empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            tc::mbar_init(&ctl.acc_full[s], 1);
            tc::mbar_init(&ctl.acc_empty[s], kEpilogueWarps);
        }
        tc::mbar_init(&ctl.done, 1);
        ctl.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpilogueWarps + kLoaderWarps) tc::tmem_alloc(&ctl.tmem, tmem_columns<T>());
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = ctl.tmem;
    if (warp < kEpilogueWarps) {
        epilogue_role<T, A_K, B_K, ACT>(g, staging, tmem, &ctl);
    } else if (warp < kEpilogueWarps + kLoaderWarps) {
        load_role<T, A_K, B_K>(g, a_ring, b_ring, &ctl);
    } else if (threadIdx.x % 32 == 0) {
        product_role<T, A_K, B_K>(g, a_ring, b_ring, tmem, &ctl);
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == kEpilogueWarps + kLoaderWarps) tc::tmem_dealloc(tmem, tmem_columns<T>());
    if (threadIdx.x == 0 && ctl.gave_up && g.status) atomicMax(g.status, static_cast<int>(NB200_ERR_WAIT_BUDGET));
}

bool multiple16(const void* p, int64_t ld, size_t size) { return aligned16(p) && (ld * size) % 16 == 0; }

}  // namespace

template <typename T, bool A_K, bool B_K, int ACT>
int mma_product(int64_t rows, int64_t cols, int64_t depth, int64_t splits, int64_t per, const T* a, int64_t as, const T* b, int64_t bs,
                const Epilogue<T>& ep, int32_t* status, cudaStream_t stream) {
    Args<T> g;
    g.a = {a, as, rows, multiple16(a, as, sizeof(T))};
    g.b = {b, bs, cols, multiple16(b, bs, sizeof(T))};
    g.rows = rows;
    g.cols = cols;
    g.depth = depth;
    g.per = per;
    g.row_tiles = ceil_div(rows, kMmaTile);
    g.col_tiles = ceil_div(cols, kMmaTile);
    g.items = g.row_tiles * g.col_tiles * splits;
    g.chunks = static_cast<int>(ceil_div(per < depth ? per : depth, kMmaChunk));
    g.ep = ep;
    g.status = status;
    const size_t wide = 4 * sizeof(T);
    auto fits = [&](const void* p) { return !p || reinterpret_cast<uintptr_t>(p) % wide == 0; };
    g.vector_out = cols % 4 == 0 && fits(ep.z) && fits(ep.y) && fits(ep.residual) && (!ep.residual || ep.ldr % 4 == 0);
    // a block keeps to one column of tiles when the grid is a multiple of their number
    int64_t grid = g.items < kSMs ? g.items : kSMs;
    g.resident = false;
    if (splits == 1 && g.chunks <= Traits<T>::b_slots && g.col_tiles <= kSMs && g.row_tiles > 1) {
        grid = kSMs / g.col_tiles * g.col_tiles;
        if (grid > g.items) grid = g.items;             // a multiple of col_tiles as well
        g.resident = true;
    }
    constexpr int smem = smem_bytes<T>();
    static_assert(smem + sizeof(Control) <= 227 * 1024, "shared memory of the product kernel");
    if (cudaFuncSetAttribute(mma_kernel<T, A_K, B_K, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return NB200_ERR_CUDA;
    mma_kernel<T, A_K, B_K, ACT><<<static_cast<unsigned>(grid), kThreads, smem, stream>>>(g);
    return launch_status();
}

#define NB200_MMA(T, A_K, B_K, ACT)                                                                                            \
    template int mma_product<T, A_K, B_K, ACT>(int64_t, int64_t, int64_t, int64_t, int64_t, const T*, int64_t, const T*, int64_t, \
                                               const Epilogue<T>&, int32_t*, cudaStream_t);
#define NB200_MMA_TYPE(T)                     \
    NB200_MMA(T, true, false, NB200_ACT_NONE) \
    NB200_MMA(T, true, false, NB200_ACT_RELU) \
    NB200_MMA(T, true, false, NB200_ACT_SILU) \
    NB200_MMA(T, true, false, NB200_ACT_GELU) \
    NB200_MMA(T, true, false, NB200_ACT_TANH) \
    NB200_MMA(T, true, true, NB200_ACT_NONE)  \
    NB200_MMA(T, false, false, NB200_ACT_NONE)
NB200_MMA_TYPE(float)
NB200_MMA_TYPE(__nv_bfloat16)
NB200_MMA_TYPE(__half)

}  // namespace nb200
