// Dense products on the 5th-generation tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// float: the tensor cores multiply 8-bit significands (bfloat16) exactly and add in 32 bits, so a float is
// cut into three bfloat16 pieces of 8 bits each, x = x0 + x1 + x2 (each piece the rounding of what the ones
// before leave: exact to 24 bits), and a product takes the six pairs of pieces whose weight is not below the
// last bit: x0y0, x0y1, x1y0, x1y1, x0y2, x2y0.  What is dropped, x1y2 + x2y1 + x2y2, is below 2^-23 |x||y|
// and 2^-26 |x||y| on average, of either sign.  (Pieces cut off instead of rounded would cost fewer
// instructions, but drop up to 2^-20, always of one sign.)  bfloat16 and half go in as they are.
//
// One persistent block per SM, warps specialised: eight loader warps bring chunks of 64 terms of both
// operands into shared memory (float: through registers, split on the way; 16-bit types: one thread issues
// tiled bulk copies, or, where rows do not start on 16-byte boundaries, all gather them), one thread issues
// the products, eight epilogue warps take finished accumulators out of tensor memory, apply bias, activation,
// residual and rounding, and send the rows off in bulk stores of whole 128-byte lines (lines written in halves or
// quarters took up to twice the time).  There are several accumulators, so the products of a tile run under the
// epilogue of the one before.  When a tile's second operand fits beside the ring of the first (the weights of a layer with
// few channels), it is loaded and split once per block and the rows stream past it.
//
// The tensor cores truncate where they add, always towards zero.  For float a chunk's products therefore go in
// order of size, the twenty small ones first, where a truncation weighs 2^-8 as much, then the four of the leading
// pieces, and the sums over chunks are formed by the epilogue warps with rounding to nearest (the running sums
// stay in tensor memory).  16-bit types have the same every 4096 terms.
//
// Measured on a B200 (copy 6548 GB/s, dense bfloat16 1651 TFLOP/s; cold L2): float, a million rows of 128 -> 128: plain
// forward 220 us = 4.9 TB/s, with silu and z kept 345 us = 4.7 TB/s, dx 177 us = 6.1 TB/s, dw 225 us = 4.8 TB/s: the
// epilogue's instructions and the shared-memory traffic of six products take turns with memory as the bound.  65,536 x
// 1024 -> 1024: 773 us = 178 TFLOP/s of float, 1.07 PFLOP/s of products (0.65).  bfloat16, a million rows of 128 -> 128:
// 86 us = 6.2 TB/s; 131,072 x 512 -> 512: 107 us, bound by L2 reads of the first operand, once per column of tiles;
// 16,384 x 4096 -> 4096: 600 us = 0.92 PFLOP/s (0.56).
#pragma once
#include <cuda.h>

#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "linear_mma.cuh"
#include "tcgen05.cuh"

namespace nb200 {
namespace {

constexpr int kEpilogueWarps = 8, kLoaderWarps = 8, kLoaders = kLoaderWarps * 32;
constexpr int kThreads = (kEpilogueWarps + kLoaderWarps + 4) * 32;   // whole warpgroups; the last has products, prefetches and two idle warps
constexpr int kLaunchRegisters = 96;                               // per thread; checked on the host
constexpr int kPieceBytes = kMmaTile * kMmaChunk * 2;              // one piece of one operand's chunk: 16 KB
constexpr int kUnits = kMmaTile * kMmaChunk / 8 / kLoaders;        // units of eight values per loader thread

// run: chunks whose products go into one accumulator.  The tensor cores cut off what they add there: measured, a sum that
// grows evenly is short by 6.3e-9 of itself per term (2^-22.2 of the sum so far with every sixteen: two additions of
// eight terms, say), always towards zero; 2^20 terms in one accumulator lost 6.6e-3, more than a bfloat16 step.  64 chunks =
// 4096 terms lose 2.5e-5, a twentieth of float16's rounding; the sums of further runs are added with rounding to nearest
// (in the columns of an accumulator, of which there is one less then).
template <typename T> struct Traits {                              // 16-bit types
    static constexpr int pieces = 1, a_slots = 4, b_slots = 8, ahead = 12, run = 64;
};
template <> struct Traits<float> {
    static constexpr int pieces = 3, a_slots = 2, b_slots = 2, ahead = 4, run = 1;
};

// What leaves: y; y and z; a product without a forward epilogue; float parts of a sum.
enum Kind { kForward, kForwardZ, kPlain, kParts };

// Registers per thread after the warpgroups have shared them out anew.  With float outputs the epilogue holds 32 columns of
// a block, and the loaders keep what they were launched with (a chunk of both float operands, or more of the values that they
// gather: dw of a million rows of 100 x 128 bfloat16 348 us, with 56 registers to a loader 448); with 16-bit outputs the
// epilogue holds twice as many columns and the loaders next to nothing.
template <typename T, int KIND>
struct Shares {
    static constexpr bool floats = sizeof(T) == 4 || KIND == kParts;
    static constexpr int epilogue = floats ? 120 : 160, loader = floats ? kLaunchRegisters : 56, product = 48;
    static_assert(kEpilogueWarps * epilogue + kLoaderWarps * loader + 4 * product <= (kEpilogueWarps + kLoaderWarps + 4) * kLaunchRegisters,
                  "registers beyond the block's own would be waited for for ever");
};

// Tensor memory: four blocks of columns, all of them accumulators or three and the running sums.
constexpr uint32_t kTmemColumns = 512;
constexpr int kSumsBlock = 3;
template <bool LONG> constexpr int buffer_count() { return LONG ? kSumsBlock : kSumsBlock + 1; }
template <typename T>
constexpr int slot_bytes() { return Traits<T>::pieces * kPieceBytes; }
template <typename T>
constexpr int smem_bytes() {
    return 1024 + (Traits<T>::a_slots + Traits<T>::b_slots) * slot_bytes<T>() + kEpilogueWarps * 4096;
}

struct Control {
    uint64_t full[8], empty[8], acc_full[4], acc_empty[4], done;
    uint32_t tmem;
    int gave_up;
    int progress;             // chunks whose products have been issued
    int odd_first, odd_last;  // float: between which items sums were not finite
};

template <typename T>
struct Operand {
    const T* p;
    int64_t ld, extent;       // row stride; rows (A) or columns (B) in all
    bool vector, wide;        // base and stride are multiples of 16, of 32 bytes
};

template <typename T>
struct Args {
    Operand<T> a, b;
    int64_t rows, cols, depth;
    int row_tiles, col_tiles, items;
    int chunks;               // chunks of a part of the sum (the last part may have fewer)
    bool resident;            // a block's second operand stays in shared memory
    bool tiled;               // operands have rows that bulk copies can address
    bool tiled_out;           // so have the outputs
    bool vector_residual, vector_bias;                   // rows of 16-byte units
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

// The units of one thread of a chunk at (m0, k0): a run of eight values of every second, fourth, ... line.  All runs
// of a thread begin at the same place of their lines, so whether they are whole is asked once; a whole run is one
// 32-byte load, or two of 16 bytes.
template <bool K_MAJOR>
struct ChunkFetch {
    using U = UnitPlace<float, K_MAJOR>;
    const float* p;
    int64_t step;
    int lines, run;           // lines left from the first on, values of a run that exist
    bool wide, vector;
    __device__ __forceinline__ ChunkFetch(const Operand<float>& o, int t, int64_t m0, int64_t k0, int64_t end) {
        const int64_t m = m0 + U::mn(t, 0), k = k0 + U::k(t, 0);
        const int64_t lines_left = K_MAJOR ? o.extent - m : end - k, run_left = K_MAJOR ? end - k : o.extent - m;
        lines = static_cast<int>(min(lines_left, int64_t(1) << 20));
        run = static_cast<int>(min(run_left, int64_t(8)));
        p = U::address(o, m, k);
        step = kLineStep * o.ld;
        wide = o.wide && run == 8;
        vector = o.vector && run == 8;
    }
    static constexpr int kLineStep = K_MAJOR ? kLoaders / 8 : kLoaders / 16;
    __device__ __forceinline__ void operator()(int q, float (&v)[8]) const {
        const float* s = p + q * step;
        const bool exists = q * kLineStep < lines;
        if (wide && exists) {
            asm volatile("ld.global.nc.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(s));
        } else if (vector && exists) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(s)), b = __ldg(reinterpret_cast<const float4*>(s) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = exists && e < run ? __ldg(s + e) : 0.f;
        }
    }
};

// Eight floats as three pieces of eight bfloat16.  What a piece leaves is exact in 32 bits and formed two at a time.
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
            if (s == 2) break;
            asm("{\n\t.reg .b64 x, y, m;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmov.b64 m, {%4, %4};\n\t"
                "fma.rn.f32x2 x, y, m, x;\n\tmov.b64 {%0, %1}, x;\n\t}"
                : "+f"(lo), "+f"(hi) : "r"(bits << 16), "r"(bits & 0xFFFF0000u), "r"(0xBF800000u));      // times -1
        }
    }
#pragma unroll
    for (int s = 0; s < 3; ++s)
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(addr + s * kPieceBytes), "r"(piece[s][0]), "r"(piece[s][1]),
                     "r"(piece[s][2]), "r"(piece[s][3]) : "memory");
}

template <typename T, bool K_MAJOR>
__device__ __forceinline__ void gather_units(const Operand<T>& o, uint32_t slot, int t, int64_t m0, int64_t k0, int64_t k_end) {
    using U = UnitPlace<T, K_MAJOR>;
#pragma unroll
    for (int q = 0; q < kUnits; ++q) {
        const int64_t m = m0 + U::mn(t, q), k = k0 + U::k(t, q);
        const int valid = U::valid(m, k, o.extent, k_end);
        const unsigned short* p = reinterpret_cast<const unsigned short*>(U::address(o, m, k));
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t lo = 2 * e < valid ? __ldg(p + 2 * e) : 0u, hi = 2 * e + 1 < valid ? __ldg(p + 2 * e + 1) : 0u;
            w[e] = lo | hi << 16;
        }
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(slot + U::offset(t, q)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                     : "memory");
    }
}

// Walks the (item, chunk) sequence of a block; every role steps through it alike.
template <typename T>
struct Walk {
    const Args<T>& g;
    int item, row_tile, col_tile, split, chunks, chunk;
    __device__ __forceinline__ explicit Walk(const Args<T>& args) : g(args), item(blockIdx.x), chunk(0) { place(); }
    __device__ __forceinline__ bool live() const { return item < g.items; }
    __device__ __forceinline__ int64_t i0() const { return int64_t(row_tile) * kMmaTile; }
    __device__ __forceinline__ int64_t j0() const { return int64_t(col_tile) * kMmaTile; }
    __device__ __forceinline__ int64_t k_begin() const { return int64_t(split) * g.chunks * kMmaChunk; }
    __device__ __forceinline__ int64_t k0() const { return k_begin() + chunk * kMmaChunk; }
    __device__ __forceinline__ int64_t k_end() const { return min(g.depth, k_begin() + int64_t(g.chunks) * kMmaChunk); }
    __device__ __forceinline__ void place() {
        if (!live()) return;
        col_tile = item % g.col_tiles;
        row_tile = item / g.col_tiles % g.row_tiles;
        split = item / g.col_tiles / g.row_tiles;
        const int64_t left = (g.depth + kMmaChunk - 1) / kMmaChunk - int64_t(split) * g.chunks;
        chunks = static_cast<int>(min(int64_t(g.chunks), left));
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

// Slot of a ring and the parity of its use; steps through the ring.
template <int SLOTS>
struct Ring {
    int slot = 0;
    unsigned parity = 0;
    bool wrapped = false;
    __device__ __forceinline__ void next() {
        if (++slot == SLOTS) {
            slot = 0;
            parity ^= 1;
            wrapped = true;
        }
    }
    // Whether slot s has been used, and the parity of its latest use.
    __device__ __forceinline__ bool used(int s, unsigned& last) const {
        last = s < slot ? parity : parity ^ 1;
        return s < slot || wrapped;
    }
};

template <typename T, bool A_K, bool B_K>
__device__ __forceinline__ void load_split(const Args<T>& g, uint32_t a_ring, uint32_t b_ring, Control* ctl) {
    // registers hold the units of the next chunk; a unit is refilled right after it has been stored
    const int t = threadIdx.x - kEpilogueWarps * 32;
    float ra[kUnits][8], rb[kUnits][8];
    Walk<T> w(g), ahead(g);
    bool with_b = true, ahead_b = true;                  // a resident operand is loaded with the block's first item
    if (!w.live()) return;
    {
        const ChunkFetch<A_K> fa(g.a, t, ahead.i0(), ahead.k0(), ahead.k_end());
        const ChunkFetch<B_K> fb(g.b, t, ahead.j0(), ahead.k0(), ahead.k_end());
#pragma unroll
        for (int q = 0; q < kUnits; ++q) {
            fa(q, ra[q]);
            fb(q, rb[q]);
        }
    }
    for (Ring<Traits<T>::a_slots> ring; w.live(); ring.next()) {
        if (ring.wrapped && !tc::mbar_wait_warp(&ctl->empty[ring.slot], ring.parity ^ 1, &ctl->gave_up)) return;
        ahead.next_chunk();
        if (g.resident && ahead.chunk == 0) ahead_b = false;
        const bool more = ahead.live();
        const uint32_t a_slot = a_ring + ring.slot * slot_bytes<T>(), b_slot = b_ring + (g.resident ? w.chunk : ring.slot) * slot_bytes<T>();
        {
            const ChunkFetch<A_K> fa(g.a, t, ahead.i0(), ahead.k0(), ahead.k_end());
#pragma unroll
            for (int q = 0; q < kUnits; ++q) {
                split_store(a_slot + UnitPlace<T, A_K>::offset(t, q), ra[q]);
                if (more) fa(q, ra[q]);
            }
        }
        if (with_b) {
            const ChunkFetch<B_K> fb(g.b, t, ahead.j0(), ahead.k0(), ahead.k_end());
#pragma unroll
            for (int q = 0; q < kUnits; ++q) {
                split_store(b_slot + UnitPlace<T, B_K>::offset(t, q), rb[q]);
                if (more && ahead_b) fb(q, rb[q]);
            }
        }
        tc::fence_smem_for_async();
        __syncwarp();
        if (threadIdx.x % 32 == 0) tc::mbar_arrive(&ctl->full[ring.slot]);
        w.next_chunk();
        if (g.resident && w.chunk == 0) with_b = false;
    }
}

// One warp walks kAhead chunks in front of the products and asks for what will be needed to be brought into L2: float
// operands (the loaders' registers hold one chunk, so they should wait for L2 and not for memory) and the rows of the
// residual (which the epilogue asks for only a block ahead).  It goes by a counter that only grows, so it may fall
// behind without missing anything, and nobody waits for it.
template <typename T, bool A_K, bool B_K, int KIND>
__device__ __forceinline__ void prefetch_role(const Args<T>& g, const void* map_a, const void* map_b, Control* ctl) {
    const int lane = threadIdx.x % 32;
    const bool operands = Traits<T>::pieces == 3 && g.tiled, residual = (KIND == kForward || KIND == kForwardZ) && g.ep.residual;
    if (!operands && !residual) return;
    const long long t0 = clock64();
    int asked = 0;
    for (Walk<T> ahead(g); ahead.live(); ahead.next_chunk(), ++asked) {
        while (asked >= *static_cast<volatile int*>(&ctl->progress) + Traits<T>::ahead) {
            if (*static_cast<volatile int*>(&ctl->gave_up) || clock64() - t0 > 64 * tc::kWaitCycles) return;
            __nanosleep(100);
        }
        if (operands && lane == 0) {
            if (A_K) tc::tile_prefetch(map_a, static_cast<int>(ahead.k0()), static_cast<int>(ahead.i0()));
            else tc::tile_prefetch(map_a, static_cast<int>(ahead.i0()), static_cast<int>(ahead.k0()));
            if (!g.resident) {
                if (B_K) tc::tile_prefetch(map_b, static_cast<int>(ahead.k0()), static_cast<int>(ahead.j0()));
                else tc::tile_prefetch(map_b, static_cast<int>(ahead.j0()), static_cast<int>(ahead.k0()));
            }
        }
        if (residual && ahead.chunk == 0) {
            const int64_t columns = min(int64_t(kMmaTile), g.cols - ahead.j0());
            for (int r = lane; r < kMmaTile && ahead.i0() + r < g.rows; r += 32) {
                const char* p = reinterpret_cast<const char*>(g.ep.residual + (ahead.i0() + r) * g.ep.ldr + ahead.j0());
                for (int64_t c = 0; c < columns * int64_t(sizeof(T)); c += 128)
                    asm volatile("prefetch.global.L2 [%0];" :: "l"(p + c));
            }
        }
    }
}

// 16-bit operands whose rows do not start on 16-byte boundaries.
template <typename T, bool A_K, bool B_K>
__device__ __forceinline__ void load_gathered(const Args<T>& g, uint32_t a_ring, uint32_t b_ring, Control* ctl) {
    const int t = threadIdx.x - kEpilogueWarps * 32;
    Walk<T> w(g);
    bool with_b = true;
    for (Ring<Traits<T>::a_slots> ring; w.live(); ring.next()) {
        const bool ok = !ring.wrapped || tc::mbar_wait(&ctl->empty[ring.slot], ring.parity ^ 1, &ctl->gave_up);
        if (ok) {
            gather_units<T, A_K>(g.a, a_ring + ring.slot * slot_bytes<T>(), t, w.i0(), w.k0(), w.k_end());
            if (with_b) gather_units<T, B_K>(g.b, b_ring + (g.resident ? w.chunk : ring.slot) * slot_bytes<T>(), t, w.j0(), w.k0(), w.k_end());
        }
        // the warp leaves together; asked behind the loads, so that nothing stands between them and the wait
        if (!__all_sync(0xFFFFFFFFu, ok)) return;
        tc::fence_smem_for_async();
        __syncwarp();
        if (threadIdx.x % 32 == 0) tc::mbar_arrive(&ctl->full[ring.slot]);
        w.next_chunk();
        if (g.resident && w.chunk == 0) with_b = false;
    }
}

// A chunk of an operand as one box of 128 rows (sum index contiguous) or two of 64 sum indices.
template <bool K_MAJOR>
__device__ __forceinline__ void load_boxes(uint32_t slot, const void* map, int64_t mn, int64_t k, uint64_t* bar) {
    if (K_MAJOR) {
        tc::tile_load(slot, map, static_cast<int>(k), static_cast<int>(mn), bar);
    } else {
        tc::tile_load(slot, map, static_cast<int>(mn), static_cast<int>(k), bar);
        tc::tile_load(slot + kPieceBytes / 2, map, static_cast<int>(mn) + 64, static_cast<int>(k), bar);
    }
}

template <typename T, bool A_K, bool B_K>
__device__ __forceinline__ void load_tiled(const Args<T>& g, const void* map_a, const void* map_b, uint32_t a_ring, uint32_t b_ring, Control* ctl) {
    Walk<T> w(g);
    bool with_b = true;
    Ring<Traits<T>::a_slots> ring;
    for (; w.live(); ring.next()) {
        if (ring.wrapped && !tc::mbar_wait(&ctl->empty[ring.slot], ring.parity ^ 1, &ctl->gave_up)) break;
        uint64_t* bar = &ctl->full[ring.slot];
        tc::mbar_expect(bar, with_b ? 2 * kPieceBytes : kPieceBytes);
        load_boxes<A_K>(a_ring + ring.slot * slot_bytes<T>(), map_a, w.i0(), w.k0(), bar);
        if (with_b) load_boxes<B_K>(b_ring + (g.resident ? w.chunk : ring.slot) * slot_bytes<T>(), map_b, w.j0(), w.k0(), bar);
        w.next_chunk();
        if (g.resident && w.chunk == 0) with_b = false;
    }
    // no copy of this thread's may be under way when the block ends, whether its products were ever formed or not
#pragma unroll 1
    for (int s = 0; s < Traits<T>::a_slots; ++s) {
        unsigned last;
        if (!ring.used(s, last)) continue;
        const uint32_t addr = tc::smem_u32(&ctl->full[s]);
        const long long t0 = clock64();
        while (!tc::mbar_try(addr, last) && clock64() - t0 < tc::kWaitCycles) {}
    }
}

template <typename T, bool A_K, bool B_K, bool LONG>
__device__ void product_role(const Args<T>& g, uint32_t a_ring, uint32_t b_ring, uint32_t tmem, Control* ctl) {
    using Tr = Traits<T>;
    constexpr int S = Tr::a_slots;
    constexpr uint32_t whole = tc::instruction_descriptor(!std::is_same<T, __half>::value, !A_K, !B_K, kMmaTile);
    constexpr uint32_t part = tc::instruction_descriptor(!std::is_same<T, __half>::value, !A_K, !B_K, kMmaTile / 2);
    constexpr uint32_t a_step = A_K ? 32 : 2048, b_step = B_K ? 32 : 2048;       // bytes from one 16-term step to the next
    Ring<S> ring;
    Ring<buffer_count<LONG>()> buffers;
    int issued = 0;
    bool ok = true;
    for (Walk<T> w(g); ok && w.live(); w.next_item()) {
        const uint32_t idesc = g.cols - w.j0() > kMmaTile / 2 ? whole : part;      // columns that do not exist are not multiplied
        for (int c = 0; ok && c < w.chunks; ++c, ring.next()) {
            const bool fresh = LONG ? c % Tr::run == 0 : c == 0, last = (LONG && (c + 1) % Tr::run == 0) || c + 1 == w.chunks;
            if (fresh && buffers.wrapped) ok = tc::mbar_wait(&ctl->acc_empty[buffers.slot], buffers.parity ^ 1, &ctl->gave_up);
            ok = ok && tc::mbar_wait(&ctl->full[ring.slot], ring.parity, &ctl->gave_up);
            if (!ok) break;
            tc::fence_after_sync();
            const uint32_t a = a_ring + ring.slot * slot_bytes<T>(), b = b_ring + (g.resident ? c : ring.slot) * slot_bytes<T>();
            const uint32_t d = tmem + buffers.slot * kMmaTile;
            bool accumulate = !fresh;
            auto products = [&](int pa, int pb) {
                const uint64_t da = tc::smem_descriptor(a + pa * kPieceBytes, A_K ? 16 : kPieceBytes / 2, 1024);
                const uint64_t db = tc::smem_descriptor(b + pb * kPieceBytes, B_K ? 16 : kPieceBytes / 2, 1024);
#pragma unroll
                for (int k = 0; k < kMmaChunk / 16; ++k) {         // the address field counts 16 bytes
                    tc::mma_f16(d, da + k * (a_step / 16), db + k * (b_step / 16), idesc, accumulate);
                    accumulate = true;
                }
            };
            if (Tr::pieces == 3) {
                products(2, 0);
                products(0, 2);
                products(1, 1);
                products(1, 0);
                products(0, 1);
            }
            products(0, 0);
            tc::commit(&ctl->empty[ring.slot]);
            *static_cast<volatile int*>(&ctl->progress) = ++issued;
            if (last) {
                tc::commit(&ctl->acc_full[buffers.slot]);
                buffers.next();
            }
        }
    }
    // nothing of this thread's may be in flight when tensor memory is given back
    tc::commit(&ctl->done);
    const uint32_t addr = tc::smem_u32(&ctl->done);
    const long long t0 = clock64();
    while (!tc::mbar_try(addr, 0) && clock64() - t0 < tc::kWaitCycles) {}
}

// 128 bytes of the output type from floats, rounded once.
__device__ __forceinline__ void pack_line(const float (&s)[32], uint32_t (&w)[32], float) {
#pragma unroll
    for (int q = 0; q < 32; ++q) w[q] = __float_as_uint(s[q]);
}
__device__ __forceinline__ void pack_line(const float (&s)[64], uint32_t (&w)[32], __nv_bfloat16) {
#pragma unroll
    for (int q = 0; q < 32; ++q) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(s[2 * q], s[2 * q + 1]);
        w[q] = *reinterpret_cast<const uint32_t*>(&r);
    }
}
__device__ __forceinline__ void pack_line(const float (&s)[64], uint32_t (&w)[32], __half) {
#pragma unroll
    for (int q = 0; q < 32; ++q) {
        const __half2 r = __floats2half2_rn(s[2 * q], s[2 * q + 1]);
        w[q] = *reinterpret_cast<const uint32_t*>(&r);
    }
}
// Half q % 2 of a word of two values, value q (0..3 or 0..7) of a 16-byte unit.
__device__ __forceinline__ float unit_value(uint32_t w, int q, __nv_bfloat16) { return __uint_as_float(q & 1 ? w & 0xFFFF0000u : w << 16); }
__device__ __forceinline__ float unit_value(uint32_t w, int q, __half) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return q & 1 ? __high2float(h) : __low2float(h);
}
__device__ __forceinline__ float unit_value(const uint32_t (&w)[4], int q, float) { return __uint_as_float(w[q]); }
template <typename T>
__device__ __forceinline__ float unit_value(const uint32_t (&w)[4], int q, T type) { return unit_value(w[q / 2], q, type); }
__device__ __forceinline__ void shared_store16(uint32_t addr, const uint32_t* w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
__device__ __forceinline__ void shared_load16(uint32_t addr, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
}

// What an epilogue warp does with blocks of 32 rows x CB columns, CB columns being 128 bytes of the output type O.
// Accumulators come out of tensor memory one row to a thread; bias, activation, residual and rounding are applied
// there, where a thread has a row's values in registers and no address to compute, and a bulk store takes the block
// from a 4 KB stage to memory, cutting off what lies outside the array.  16-byte unit u of row r of the stage is at
// unit u ^ (r % 8): the order of the bulk store's 128-byte swizzle, and free of bank conflicts.
template <typename T, typename O, int ACT, int KIND>
struct Writer {
    static constexpr int CB = 128 / sizeof(O), U = 16 / sizeof(O);           // columns of a block, of a unit
    const Args<T>& g;
    const void *map_y, *map_z;
    const uint32_t stage;
    const int lane;

    __device__ __forceinline__ Writer(const Args<T>& args, const void* my, const void* mz, uint32_t s)
        : g(args), map_y(my), map_z(mz), stage(s), lane(threadIdx.x % 32) {}
    __device__ __forceinline__ uint32_t place(int r, int u) const { return stage + r * 128 + ((u ^ (r & 7)) * 16); }

    // Eight lanes read a row's 128 bytes, a warp four rows at a time; asked for early, so that the way overlaps.
    __device__ __forceinline__ void fetch_residual(int64_t row0, int64_t col0, uint32_t (&next)[8][4]) const {
        const int64_t i = row0 + lane / 8, j = col0 + lane % 8 * U;
        const int count = j < g.cols ? static_cast<int>(min(int64_t(8), (g.rows - i + 3) / 4)) : 0;
        const T* p = g.ep.residual + i * g.ep.ldr + j;
#pragma unroll
        for (int e = 0; e < 8; ++e, p += 4 * g.ep.ldr)
            if (e < count) {
                const uint4 u = *reinterpret_cast<const uint4*>(p);
                next[e][0] = u.x; next[e][1] = u.y; next[e][2] = u.z; next[e][3] = u.w;
            }
    }
    // The stage may be written: the last store has read it.
    __device__ __forceinline__ void open() const {
        if (g.tiled_out && lane == 0) tc::stores_read();
        __syncwarp();
    }
    // This thread's row of the block to the stage, and from there to memory.
    __device__ __forceinline__ void close(const float (&s)[CB], O* base, const void* map, int split, int64_t row0, int64_t col0) const {
        uint32_t w[32];
        pack_line(s, w, O());
        send(w, base, map, split, row0, col0);
    }
    __device__ __forceinline__ void send(const uint32_t (&w)[32], O* base, const void* map, int split, int64_t row0, int64_t col0) const {
#pragma unroll
        for (int u = 0; u < 8; ++u) shared_store16(place(lane, u), w + 4 * u);
        if (g.tiled_out) {
            tc::fence_smem_for_async();
            __syncwarp();
            if (lane == 0) tc::tile_store(map, static_cast<int>(col0), static_cast<int>(row0), split, stage);
        } else {                                     // rows that start anywhere: a lane per column
            __syncwarp();
            const int rows = static_cast<int>(min(int64_t(32), g.rows - row0));
#pragma unroll 1
            for (int c = lane; c < CB && col0 + c < g.cols; c += 32) {
                O* out = base + (split * g.rows + row0) * g.cols + col0 + c;
#pragma unroll 4
                for (int r = 0; r < rows; ++r, out += g.cols) {
                    const uint32_t addr = place(r, c / U) + c % U * sizeof(O);
                    if constexpr (sizeof(O) == 4) {
                        float v;
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
                        *out = v;
                    } else {
                        unsigned short v;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
                        *reinterpret_cast<unsigned short*>(out) = v;
                    }
                }
            }
        }
    }

    __device__ __forceinline__ void block(float (&v)[CB], int split, int64_t row0, int64_t col0, const uint32_t (&next)[8][4]) const {
        const Epilogue<T>& ep = g.ep;
        if constexpr (KIND == kParts) {
            open();
            close(v, ep.partial, map_y, split, row0, col0);
        } else if constexpr (KIND == kPlain) {
            open();
            close(v, ep.y, map_y, 0, row0, col0);
        } else {
            if (ep.bias) {
                if (g.vector_bias && col0 + CB <= g.cols) {
#pragma unroll
                    for (int u = 0; u < CB; u += U) {
                        const uint4 b4 = *reinterpret_cast<const uint4*>(ep.bias + col0 + u);
                        const uint32_t b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                        for (int q = 0; q < U; q += 2)
                            (Pair(v[u + q], v[u + q + 1]) + Pair(unit_value(b, q, O()), unit_value(b, q + 1, O()))).to(v[u + q], v[u + q + 1]);
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < CB; ++q) v[q] += col0 + q < g.cols ? to_acc(ep.bias[col0 + q]) : 0.f;
                }
            }
            if constexpr (KIND == kForwardZ) {
                open();
                if constexpr (ACT == NB200_ACT_RELU && sizeof(T) == 2) {   // relu's slope needs more than the rounded value
                    float t[CB];
#pragma unroll
                    for (int q = 0; q < CB; ++q) t[q] = to_acc(rounded_z<T, ACT>(v[q]));
                    close(t, ep.z, map_z, 0, row0, col0);
                } else if constexpr (slope_has_z<ACT>() && sizeof(T) == 2) {
                    uint32_t w[32];
                    pack_line(v, w, O());
                    float most = 0.f;
#pragma unroll
                    for (int q = 0; q < CB; ++q) most = fmaxf(most, fabsf(v[q]));
                    if (most > largest_finite<T>())          // hardly ever; the bits of the largest number are those of infinity less one
#pragma unroll
                        for (int q = 0; q < CB; ++q)
                            if (isfinite(v[q]) && isinf(unit_value(w[q / 2], q, O()))) w[q / 2] -= q & 1 ? 0x10000u : 1u;
                    send(w, ep.z, map_z, 0, row0, col0);
                } else {
                    close(v, ep.z, map_z, 0, row0, col0);
                }
            }
#pragma unroll
            for (int q = 0; q < CB; q += 2) activate_pair<ACT>(v[q], v[q + 1]);
            open();
            if (ep.residual) {
                if (g.vector_residual) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) shared_store16(place(lane / 8 + 4 * e, lane % 8), next[e]);
                    __syncwarp();
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        uint32_t r[4];
                        shared_load16(place(lane, u), r);
#pragma unroll
                        for (int q = 0; q < U; q += 2)
                            (Pair(v[u * U + q], v[u * U + q + 1]) + Pair(unit_value(r, q, O()), unit_value(r, q + 1, O())))
                                .to(v[u * U + q], v[u * U + q + 1]);
                    }
                } else if (row0 + lane < g.rows) {
                    const T* p = ep.residual + (row0 + lane) * ep.ldr + col0;
#pragma unroll
                    for (int q = 0; q < CB; ++q)
                        if (col0 + q < g.cols) v[q] += to_acc(p[q]);
                }
            }
            close(v, ep.y, map_y, 0, row0, col0);
        }
    }
};

// The accumulators of one item (float: one per chunk).
template <bool LONG, typename T, typename O, int ACT, int KIND>
__device__ __forceinline__ bool epilogue_item(const Args<T>& g, const Walk<T>& w, const Writer<T, O, ACT, KIND>& out,
                                              Ring<buffer_count<LONG>()>& buffers, uint32_t tmem, Control* ctl) {
    using Tr = Traits<T>;
    constexpr int CB = Writer<T, O, ACT, KIND>::CB;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int quarter = warp % 4, half = warp / 4;                 // tensor memory lanes and columns of this warp
    const int64_t row0 = w.i0() + quarter * 32, col0 = w.j0() + half * 64;
    auto present = [&](int block) { return row0 < g.rows && col0 + block * CB < g.cols; };
    const uint32_t mine = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * 64;
    const uint32_t sums = mine + kSumsBlock * kMmaTile;
    auto arrived = [&]() {
        if (!tc::mbar_wait_warp(&ctl->acc_full[buffers.slot], buffers.parity, &ctl->gave_up)) return false;
        tc::fence_after_sync();
        return true;
    };
    auto release = [&]() {                                         // everything has left the accumulator
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&ctl->acc_empty[buffers.slot]);
        buffers.next();
    };
    const int parts = LONG ? (w.chunks + Tr::run - 1) / Tr::run : 1;
    if constexpr (LONG) {
#pragma unroll 1
        for (int part = 0; part + 1 < parts; ++part) {
            if (!arrived()) return false;
            const uint32_t from = mine + buffers.slot * kMmaTile;
#pragma unroll 2
            for (int c = 0; c < 64 && present(c / CB); c += 16) {
                float v[16], sum[16];
                tc::tmem_load16(from + c, v);
                if (part > 0) tc::tmem_load16(sums + c, sum);
                tc::tmem_wait16(v);
                if (part > 0) {
                    tc::tmem_wait16(sum);
#pragma unroll
                    for (int q = 0; q < 16; q += 2) (Pair(v[q], v[q + 1]) + Pair(sum[q], sum[q + 1])).to(v[q], v[q + 1]);
                }
                tc::tmem_store16(sums + c, v);
            }
            tc::tmem_stores_done();
            release();
        }
    }
    if (!arrived()) return false;
    const uint32_t from = mine + buffers.slot * kMmaTile;
#pragma unroll 1
    for (int block = 0; block < 64 / CB; ++block) {
        if (!present(block)) break;
        const int64_t col = col0 + block * CB;
        uint32_t residual[8][4];
        if ((KIND == kForward || KIND == kForwardZ) && g.ep.residual && g.vector_residual) out.fetch_residual(row0, col, residual);
        float v[CB];
#pragma unroll
        for (int q = 0; q < CB; q += 16) tc::tmem_load16(from + block * CB + q, *reinterpret_cast<float(*)[16]>(v + q));
        if (LONG && parts > 1) {
#pragma unroll
            for (int h = 0; h < CB; h += 16) {
                float sum[16];
                tc::tmem_load16(sums + block * CB + h, sum);
                tc::tmem_wait16(v + h);
                tc::tmem_wait16(sum);
#pragma unroll
                for (int q = 0; q < 16; q += 2)
                    (Pair(v[h + q], v[h + q + 1]) + Pair(sum[q], sum[q + 1])).to(v[h + q], v[h + q + 1]);
            }
        } else {
#pragma unroll
            for (int q = 0; q < CB; q += 16) tc::tmem_wait16(v + q);
        }
        if (block + 1 == 64 / CB || !present(block + 1)) release();
        if constexpr (Tr::pieces == 3) {
            Pair zeros = both(0.f);                                // NaN if any of the values is not finite
#pragma unroll
            for (int q = 0; q < CB; q += 2) zeros = fma(Pair(v[q], v[q + 1]), both(0.f), zeros);
            float t, t2;
            zeros.to(t, t2);
            t += t2;
            if (t != t && row0 + lane < g.rows) {                  // left as it is for now; see form_again
                atomicMin(&ctl->odd_first, w.item);
                atomicMax(&ctl->odd_last, w.item);
            }
            __syncwarp();
            // the values are settled before bias and residual are called for (left to the compiler, 27 registers go to memory)
#pragma unroll
            for (int q = 0; q < CB; ++q) asm volatile("" : "+f"(v[q]));
        }
        out.block(v, w.split, row0, col, residual);
    }
    if (!present(0)) release();
    return true;
}

template <bool LONG, typename T, int ACT, int KIND>
__device__ __forceinline__ void epilogue_role(const Args<T>& g, const void* map_y, const void* map_z, uint32_t staging, uint32_t tmem,
                                              Control* ctl) {
    using O = typename std::conditional<KIND == kParts, float, T>::type;
    const int warp = threadIdx.x / 32;
    const Writer<T, O, ACT, KIND> out(g, map_y, map_z, staging + warp * 4096);
    Ring<buffer_count<LONG>()> buffers;
    Walk<T> w(g);
    for (bool ok = true; ok && w.live(); w.next_item()) ok = epilogue_item<LONG, T, O, ACT, KIND>(g, w, out, buffers, tmem, ctl);
    if (threadIdx.x % 32 == 0) tc::stores_done();
}

// Float sums again in plain 32-bit arithmetic: the pieces of an infinity, or of a value that rounds to one in 16 bits,
// make a NaN where the product may be neither.  Either the lanes of a warp share the terms of one value (128 at a time),
// or each has the value of its own row (eight terms at a time): whichever takes fewer trips to memory for the `count`
// values of a column.  A sum that is NaN stays so and ends early.
template <typename T, bool A_K, bool B_K>
struct Plain {
    const Args<T>& g;
    const int64_t k_begin, k_end;
    __device__ __forceinline__ float a(int64_t i, int64_t k) const { return to_acc(A_K ? g.a.p[i * g.a.ld + k] : g.a.p[k * g.a.ld + i]); }
    __device__ __forceinline__ float b(int64_t k, int64_t j) const { return to_acc(B_K ? g.b.p[j * g.b.ld + k] : g.b.p[k * g.b.ld + j]); }
    __device__ __forceinline__ bool share_terms(int count) const {
        const int64_t terms = k_end - k_begin;
        return count * ((terms + 127) / 128) <= (terms + 7) / 8;
    }
    // The value at (i, j), the same for all lanes.
    __device__ __forceinline__ float shared(int64_t i, int64_t j) const {
        const int lane = threadIdx.x % 32;
        float v = 0.f;
#pragma unroll 1
        for (int64_t k = k_begin + lane; k - lane < k_end; k += 128) {
            float x[4], y[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {                              // without conditions: the loads go out together
                const int64_t there = min(k + 32 * u, k_end - 1);
                x[u] = a(i, there);
                y[u] = b(there, j);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) v = k + 32 * u < k_end ? fmaf(x[u], y[u], v) : v;
            if (__any_sync(0xFFFFFFFFu, isnan(v))) break;
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
        return v;
    }
    // The value at (i, j) of every lane that wants one; j is the same for all.
    __device__ __forceinline__ float own(int64_t i, int64_t j, bool wanted) const {
        float v = 0.f;
        i = min(i, g.rows - 1);
#pragma unroll 1
        for (int64_t k = k_begin; k < k_end; k += 8) {
            float x[8], y[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int64_t there = min(k + u, k_end - 1);
                x[u] = a(i, there);
                y[u] = b(there, j);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) v = k + u < k_end ? fmaf(x[u], y[u], v) : v;
            if (__all_sync(0xFFFFFFFFu, !wanted || isnan(v))) break;
        }
        return v;
    }
};

// Forms again what is not finite of the items among which the epilogue has met such sums.  It runs when everything else
// of the block is done, so nobody waits for it however long the sums are.  Its eight warps take pieces of 32 x 32 values,
// a row to a lane.  Measured, forward, dx and dw of a million rows of 128 floats, 0.66 ms: 2.6 ms with one infinity in x
// (128 sums of 7000 terms), 39 ms with a row of them (every entry of dw), 12 ms with nothing but NaN.
template <typename T, bool A_K, bool B_K, int ACT, int KIND>
__device__ __noinline__ void form_again(const Args<T>& g, const Control* ctl) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int first = ctl->odd_first, last = ctl->odd_last;
    for (Walk<T> w(g); w.live() && w.item <= last; w.next_item()) {
        if (w.item < first) continue;
        const Plain<T, A_K, B_K> plain{g, w.k_begin(), w.k_end()};
        for (int piece = warp; piece < 16; piece += kEpilogueWarps) {
            const int64_t i = w.i0() + piece % 4 * 32 + lane, j0 = w.j0() + piece / 4 * 32;
            for (int64_t j = j0; j < j0 + 32 && j < g.cols; ++j) {
                const int64_t e = i * g.cols + j;
                float* part = KIND == kParts ? g.ep.partial + w.split * g.rows * g.cols + e : nullptr;
                bool wanted = false;
                if (i < g.rows) {
                    const float seen = KIND == kParts ? *part : to_acc(KIND == kForwardZ ? g.ep.z[e] : g.ep.y[e]);
                    wanted = !isfinite(seen);
                }
                unsigned left = __ballot_sync(0xFFFFFFFFu, wanted);
                if (left == 0) continue;
                float v = 0.f;
                if (plain.share_terms(__popc(left))) {
#pragma unroll 1
                    for (; left != 0; left &= left - 1) {
                        const int row = __ffs(left) - 1;
                        const float again = plain.shared(i - lane + row, j);
                        if (lane == row) v = again;
                    }
                } else {
                    v = plain.own(i, j, wanted);
                }
                if (!wanted) continue;
                if constexpr (KIND == kParts) {
                    *part = v;
                } else if constexpr (KIND == kPlain) {
                    g.ep.y[e] = from_acc<T>(v);
                } else {
                    if (g.ep.bias) v += to_acc(g.ep.bias[j]);
                    if constexpr (KIND == kForwardZ) g.ep.z[e] = rounded_z<T, ACT>(v);
                    v = activate<ACT>(v);
                    if (g.ep.residual) v += to_acc(g.ep.residual[i * g.ep.ldr + j]);
                    g.ep.y[e] = from_acc<T>(v);
                }
            }
        }
    }
}

// After a wait that ran out: NaN over all that this block was to write, so that nothing passes for a result.  The
// epilogue warps do it, once all stores are done: the others have given registers away.  Out of line, so that the
// roles' registers are not shared out with it in mind (gathered dw of a million rows of 100 x 128 bfloat16 398 us, inline 488 at the time).
template <typename T, typename O>
__device__ __noinline__ void write_nan(const Args<T>& g, O* out) {
    for (Walk<T> w(g); w.live(); w.next_item()) {
        const int64_t columns = min(int64_t(kMmaTile), g.cols - w.j0()), rows = min(int64_t(kMmaTile), g.rows - w.i0());
        O* corner = out + (w.split * g.rows + w.i0()) * g.cols + w.j0();
        for (int e = threadIdx.x; e < rows * columns; e += kEpilogueWarps * 32) corner[e / columns * g.cols + e % columns] = from_acc<O>(NAN);
    }
}

template <typename T, bool A_K, bool B_K, int ACT, int KIND, bool LONG>
__global__ void __launch_bounds__(kThreads, 1) mma_kernel(const __grid_constant__ Args<T> g,
                                                          const __grid_constant__ CUtensorMap map_a,
                                                          const __grid_constant__ CUtensorMap map_b,
                                                          const __grid_constant__ CUtensorMap map_y,
                                                          const __grid_constant__ CUtensorMap map_z) {
    using Tr = Traits<T>;
    using Share = Shares<T, KIND>;
    extern __shared__ char raw[];
    __shared__ Control ctl;
    const uint32_t base = (tc::smem_u32(raw) + 1023) / 1024 * 1024;
    const uint32_t a_ring = base, b_ring = a_ring + Tr::a_slots * slot_bytes<T>(), staging = b_ring + Tr::b_slots * slot_bytes<T>();
    const int warp = threadIdx.x / 32;
    if (threadIdx.x == 0) {
        for (int s = 0; s < Tr::a_slots; ++s) {
            tc::mbar_init(&ctl.full[s], Tr::pieces == 1 && g.tiled ? 1 : kLoaderWarps);
            tc::mbar_init(&ctl.empty[s], 1);
        }
        for (int s = 0; s < buffer_count<LONG>(); ++s) {
            tc::mbar_init(&ctl.acc_full[s], 1);
            tc::mbar_init(&ctl.acc_empty[s], kEpilogueWarps);
        }
        tc::mbar_init(&ctl.done, 1);
        ctl.gave_up = 0;
        ctl.progress = 0;
        ctl.odd_first = INT_MAX;
        ctl.odd_last = -1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpilogueWarps + kLoaderWarps) tc::tmem_alloc(&ctl.tmem, kTmemColumns);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = ctl.tmem;
    if (warp < kEpilogueWarps) {
        tc::registers_up<Share::epilogue>();
        epilogue_role<LONG, T, ACT, KIND>(g, &map_y, &map_z, staging, tmem, &ctl);
    } else if (warp < kEpilogueWarps + kLoaderWarps) {
        if constexpr (Share::loader < kLaunchRegisters) tc::registers_down<Share::loader>();
        if constexpr (Tr::pieces == 3) tc::registers_up<Share::loader>();    // as many as it has: without it the compiler spills
        if constexpr (Tr::pieces == 3) {
            load_split<T, A_K, B_K>(g, a_ring, b_ring, &ctl);
        } else {
            if (!g.tiled)
                load_gathered<T, A_K, B_K>(g, a_ring, b_ring, &ctl);
            else if (threadIdx.x == kEpilogueWarps * 32)
                load_tiled<T, A_K, B_K>(g, &map_a, &map_b, a_ring, b_ring, &ctl);
        }
    } else {
        tc::registers_down<Share::product>();
        if (threadIdx.x == (kEpilogueWarps + kLoaderWarps) * 32) product_role<T, A_K, B_K, LONG>(g, a_ring, b_ring, tmem, &ctl);
        if (warp == kEpilogueWarps + kLoaderWarps + 1) prefetch_role<T, A_K, B_K, KIND>(g, &map_a, &map_b, &ctl);
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == kEpilogueWarps + kLoaderWarps) tc::tmem_dealloc(tmem, kTmemColumns);
    if constexpr (Tr::pieces == 3)
        if (ctl.odd_last >= 0 && warp < kEpilogueWarps) {
            asm volatile("fence.proxy.async;" ::: "memory");         // the bulk stores are done; what they wrote is read
            form_again<T, A_K, B_K, ACT, KIND>(g, &ctl);
        }
    if (ctl.gave_up && warp < kEpilogueWarps) {
        if (threadIdx.x == 0 && g.status) atomicMax(g.status, static_cast<int>(NB200_ERR_WAIT_BUDGET));
        if constexpr (KIND == kParts) write_nan<T, float>(g, g.ep.partial);
        else write_nan<T, T>(g, g.ep.y);
        if constexpr (KIND == kForwardZ) write_nan<T, T>(g, g.ep.z);
    }
}

bool multiple_of(size_t bytes, const void* p, int64_t ld, size_t size) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (ld * size) % bytes == 0;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// Boxes of `lines` rows of a [outer, inner] array with row stride ld: 64 contiguous 16-bit values in the tensor
// cores' order, or the floats of a whole chunk.
template <typename T>
bool make_map(CUtensorMap* map, const T* p, int64_t inner, int64_t outer, int64_t ld, int lines) {
    constexpr bool split = std::is_same<T, float>::value;
    const EncodeTiled encode = encode_tiled();
    if (!encode || inner > INT32_MAX || outer > INT32_MAX || ld * int64_t(sizeof(T)) >= (int64_t(1) << 40)) return false;
    const cuuint64_t size[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    const cuuint64_t stride[1] = {static_cast<cuuint64_t>(ld) * sizeof(T)};
    const cuuint32_t box[2] = {split ? static_cast<cuuint32_t>(kMmaTile * kMmaChunk / lines) : kMmaChunk, static_cast<cuuint32_t>(lines)};
    const cuuint32_t step[2] = {1, 1};
    const CUtensorMapDataType type = split ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                           : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode(map, type, 2, const_cast<T*>(p), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  split ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Boxes of 32 rows by 128 bytes of a [parts, rows, cols] array, for the epilogue's stores.
template <typename O>
bool make_output_map(CUtensorMap* map, O* p, int64_t rows, int64_t cols, int64_t parts) {
    const EncodeTiled encode = encode_tiled();
    const uint64_t line = static_cast<uint64_t>(cols) * sizeof(O), part = static_cast<uint64_t>(rows) * line;
    if (!encode || !aligned16(p) || line % 16 != 0 || rows > INT32_MAX || cols > INT32_MAX || part >= (uint64_t(1) << 40)) return false;
    const cuuint64_t size[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(parts)};
    const cuuint64_t stride[2] = {line, part};
    const cuuint32_t box[3] = {128 / sizeof(O), 32, 1}, step[3] = {1, 1, 1};
    const CUtensorMapDataType type = sizeof(O) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    return encode(map, type, 3, p, size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool A_K, bool B_K, int ACT, int KIND, bool LONG>
int launch_kernel(const Args<T>& g, const CUtensorMap& map_a, const CUtensorMap& map_b, const CUtensorMap& map_y, const CUtensorMap& map_z,
                  unsigned grid, int smem, cudaStream_t stream) {
    // once per kernel and device
    static std::atomic<uint64_t> prepared{0};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return NB200_ERR_CUDA;
    if (device >= 64 || !(prepared.load(std::memory_order_acquire) >> device & 1)) {
        cudaFuncAttributes attr;
        if (cudaFuncSetAttribute(mma_kernel<T, A_K, B_K, ACT, KIND, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
            cudaFuncGetAttributes(&attr, mma_kernel<T, A_K, B_K, ACT, KIND, LONG>) != cudaSuccess)
            return NB200_ERR_CUDA;
        if (attr.numRegs != kLaunchRegisters) return NB200_ERR_PRECONDITION;
        if (device < 64) prepared.fetch_or(uint64_t(1) << device, std::memory_order_release);
    }
    mma_kernel<T, A_K, B_K, ACT, KIND, LONG><<<grid, kThreads, smem, stream>>>(g, map_a, map_b, map_y, map_z);
    return launch_status();
}

template <typename T, bool A_K, bool B_K, int ACT, int KIND>
int launch(int64_t rows, int64_t cols, int64_t depth, int64_t splits, int64_t per, const T* a, int64_t as, const T* b, int64_t bs,
                const Epilogue<T>& ep, int32_t* status, cudaStream_t stream) {
    const int64_t row_tiles = ceil_div(rows, kMmaTile), col_tiles = ceil_div(cols, kMmaTile);
    if (row_tiles > INT32_MAX || col_tiles > INT32_MAX || row_tiles * col_tiles > INT32_MAX / 2 ||
        row_tiles * col_tiles * splits > INT32_MAX / 2)
        return NB200_ERR_TOO_LARGE;
    Args<T> g;
    g.a = {a, as, rows, multiple_of(16, a, as, sizeof(T)), multiple_of(32, a, as, sizeof(T))};
    g.b = {b, bs, cols, multiple_of(16, b, bs, sizeof(T)), multiple_of(32, b, bs, sizeof(T))};
    g.rows = rows;
    g.cols = cols;
    g.depth = depth;
    g.row_tiles = static_cast<int>(row_tiles);
    g.col_tiles = static_cast<int>(col_tiles);
    g.items = static_cast<int>(row_tiles * col_tiles * splits);
    g.chunks = static_cast<int>(ceil_div(per < depth ? per : depth, kMmaChunk));
    g.ep = ep;
    g.status = status;
    CUtensorMap map_a{}, map_b{}, map_y{}, map_z{};
    g.tiled_out = KIND == kParts ? make_output_map(&map_y, ep.partial, rows, cols, splits)
                                 : make_output_map(&map_y, ep.y, rows, cols, 1) && (!ep.z || make_output_map(&map_z, ep.z, rows, cols, 1));
    g.vector_residual = (cols * sizeof(T)) % 16 == 0 && multiple_of(16, ep.residual, ep.ldr, sizeof(T));
    g.vector_bias = aligned16(ep.bias);
    // 16-bit types: boxes that the tensor cores read; float: boxes for the prefetches
    g.tiled = g.a.vector && g.b.vector &&
              (A_K ? make_map(&map_a, a, depth, rows, as, kMmaTile) : make_map(&map_a, a, rows, depth, as, kMmaChunk)) &&
              (B_K ? make_map(&map_b, b, depth, cols, bs, kMmaTile) : make_map(&map_b, b, cols, depth, bs, kMmaChunk));
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
    if (Traits<T>::pieces == 3 || g.chunks > Traits<T>::run)
        return launch_kernel<T, A_K, B_K, ACT, KIND, true>(g, map_a, map_b, map_y, map_z, static_cast<unsigned>(grid), smem, stream);
    if constexpr (Traits<T>::pieces == 1)
        return launch_kernel<T, A_K, B_K, ACT, KIND, false>(g, map_a, map_b, map_y, map_z, static_cast<unsigned>(grid), smem, stream);
    return NB200_ERR_BAD_ARG;                            // not reached
}

}  // namespace

template <typename T, bool A_K, bool B_K, int ACT>
int mma_product(int64_t rows, int64_t cols, int64_t depth, int64_t splits, int64_t per, const T* a, int64_t as, const T* b, int64_t bs,
                const Epilogue<T>& ep, int32_t* status, cudaStream_t stream) {
    if constexpr (!A_K) {
        return launch<T, A_K, B_K, ACT, kParts>(rows, cols, depth, splits, per, a, as, b, bs, ep, status, stream);
    } else if constexpr (B_K) {
        return launch<T, A_K, B_K, ACT, kPlain>(rows, cols, depth, splits, per, a, as, b, bs, ep, status, stream);
    } else {
        return ep.z ? launch<T, A_K, B_K, ACT, kForwardZ>(rows, cols, depth, splits, per, a, as, b, bs, ep, status, stream)
                    : launch<T, A_K, B_K, ACT, kForward>(rows, cols, depth, splits, per, a, as, b, bs, ep, status, stream);
    }
}

#define NB200_MMA(T, A_K, B_K, ACT)                                                                                            \
    template int mma_product<T, A_K, B_K, ACT>(int64_t, int64_t, int64_t, int64_t, int64_t, const T*, int64_t, const T*, int64_t, \
                                               const Epilogue<T>&, int32_t*, cudaStream_t);
// The three products of a layer in one type: forward with every activation, dx, dw.
#define NB200_MMA_TYPE(T)                     \
    NB200_MMA(T, true, false, NB200_ACT_NONE) \
    NB200_MMA(T, true, false, NB200_ACT_RELU) \
    NB200_MMA(T, true, false, NB200_ACT_SILU) \
    NB200_MMA(T, true, false, NB200_ACT_GELU) \
    NB200_MMA(T, true, false, NB200_ACT_TANH) \
    NB200_MMA(T, true, true, NB200_ACT_NONE)  \
    NB200_MMA(T, false, false, NB200_ACT_NONE)

}  // namespace nb200
