// INT8 x INT8 matrix product: activations quantized per row, weights per
// column, exact 32-bit integer sums on v_mfma_i32_32x32x32_i8.
//
//   C[m, n] = fp32(sum_k a[m, k] w[k, n]) * (a_scale[m] * w_scale[n])
//
// Both operands lie in blocks of 32 rows (columns) x 64 k, 2 KB each: 16-byte
// chunk kc * 32 + r holds row r's k = 16 kc .. + 15 (kc 0..3), so a wave reads
// the operand of one MFMA (32 rows x 32 k: lane l row l % 32, k 16 (l / 32) ..
// + 15) as 1 KB of adjacent bytes.  A panel of 32 columns is contiguous along
// k.  Rows and columns are padded to 32 (padding is read, never used), k to 64
// with zeros.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>

#include "kv_q8.h"
#include "vm_device.h"
#include "vm_internal.h"

namespace vmhip {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kT = 256;
constexpr int kBlockBytes = 2048;
constexpr int kMaxTiles = 512;           // tiles that several workgroups may share
constexpr int kTicketStride = 16;        // a ticket has a 64-byte line of its own
constexpr int64_t kTicketBytes = kMaxTiles * kTicketStride * 4;
constexpr int kMaxSplits = 16;

int64_t blocks32(int64_t x) { return (x + 31) / 32; }
int64_t steps64(int64_t k) { return (k + 63) / 64; }
int64_t staged_codes(int64_t rows, int64_t k) { return blocks32(rows) * steps64(k) * kBlockBytes; }

// ---- Weights: thread (column, 16-k chunk) gathers 16 bytes of its column;
// 32 lanes read 32 adjacent bytes of a row and write 512 adjacent ones.
__global__ __launch_bounds__(kT) void a8_pack_kernel(const int8_t* __restrict__ w, int8_t* __restrict__ out, int64_t k,
                                                     int64_t n, int64_t steps, int64_t chunks) {
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * kT + threadIdx.x; u < chunks;
         u += static_cast<int64_t>(gridDim.x) * kT) {
        const int64_t block = u >> 7;          // (panel, step)
        const int c = static_cast<int>(u & 127);
        const int64_t col = block / steps * 32 + (c & 31);
        const int64_t k0 = block % steps * 64 + (c >> 5) * 16;
        alignas(16) int8_t e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = col < n && k0 + i < k ? w[(k0 + i) * n + col] : int8_t(0);
        *reinterpret_cast<u32x4*>(out + u * 16) = *reinterpret_cast<const u32x4*>(e);
    }
}

// ---- Activations: a workgroup a row, 16 adjacent values a lane and chunk, read
// once (the first kHeld chunks of a lane wait in registers for the maximum).
// 16 x 2048 fp32 3.1 us, 512 x 2048 3.3-4.8, 2048 x 8192 bf16 19-21 (50 MB: 2.5 TB/s.
// About 20 VALU instructions a value, the rounding half away from zero among them,
// are 10 us of it, and a row's loads, maximum and stores follow one another; with
// codes gathered in LDS, so that 64 adjacent bytes are written instead of 16, it
// took as long there and half as long again at 512 rows).
template <typename T>
__device__ __forceinline__ void load16(const T* p, int valid, float (&x)[16]);
template <>
__device__ __forceinline__ void load16<float>(const float* p, int valid, float (&x)[16]) {
    if (valid >= 16) {
        __builtin_memcpy(x, p, 64);
    } else {
        p = apart(p);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = i < valid ? p[i] : 0.0f;
    }
}
template <bool kBf16>
__device__ __forceinline__ void load16_half(const uint16_t* p, int valid, float (&x)[16]) {
    uint16_t h[16];
    if (valid >= 16) {
        __builtin_memcpy(h, p, 32);
    } else {
        p = apart(p);
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = i < valid ? p[i] : uint16_t(0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
        x[i] = kBf16 ? __uint_as_float(static_cast<uint32_t>(h[i]) << 16)
                     : static_cast<float>(__builtin_bit_cast(_Float16, h[i]));
}
template <>
__device__ __forceinline__ void load16<F16>(const F16* p, int valid, float (&x)[16]) {
    load16_half<false>(&p->bits, valid, x);
}
template <>
__device__ __forceinline__ void load16<BF16>(const BF16* p, int valid, float (&x)[16]) {
    load16_half<true>(&p->bits, valid, x);
}

constexpr int kHeld = 4;   // chunks of a lane kept in registers between the two passes

template <typename T>
__global__ __launch_bounds__(kT) void a8_stage_row_kernel(const T* __restrict__ a, int8_t* __restrict__ out,
                                                          float* __restrict__ scales, int64_t rows, int k, int steps,
                                                          int spread) {
    __shared__ uint32_t wave_max[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // Workgroups go to the XCDs in turn; the 32 rows of a block, whose codes
    // share lines, to one of them (rows of 256 at a time): staging and product
    // of 512 x 2048 x 5632 20.3 -> 19.7 us, of 1000 rows 30.4 -> 29.2.
    int64_t row = blockIdx.x;
    if (spread) row = (row & ~int64_t(255)) | (row & 7) << 5 | (row & 255) >> 3;
    if (row >= rows) return;
    const int chunks = steps * 4;
    const T* src = a + row * k;
    float x[kHeld][16];
    uint32_t m = 0;
    for (int c = threadIdx.x, u = 0; c < chunks; c += kT, ++u) {
        float y[16];
        load16(src + c * 16, k - c * 16, y);
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (h == u)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[h][i] = y[i];
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), s, 64)));
    if (lane == 0) wave_max[wave] = m;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 4; ++v) m = max(m, wave_max[v]);
    const Q8Scale q8 = q8_scale(m);
    int8_t* dst = out + (row >> 5) * steps * kBlockBytes + (row & 31) * 16;
    for (int c = threadIdx.x, u = 0; c < chunks; c += kT, ++u) {
        float y[16];
        if (u < kHeld) {
#pragma unroll
            for (int h = 0; h < kHeld; ++h)
                if (h == u)
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = x[h][i];
        } else {
            load16(src + c * 16, k - c * 16, y);
        }
        alignas(16) int8_t e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = q8_code(y[i], q8.inv);
        *reinterpret_cast<u32x4*>(dst + (c >> 2) * static_cast<int64_t>(kBlockBytes) + (c & 3) * 512) =
            *reinterpret_cast<const u32x4*>(e);
    }
    if (threadIdx.x == 0) scales[row] = q8.scale;
}

// ---- The product.
struct Args {
    const int8_t* a;
    const float* a_scale;
    const int8_t* w;
    const float* w_scale;
    void* c;
    unsigned* tickets;
    int* parts;
    int64_t rows, n;
    int row_blocks, steps, panels, tiles_m, splits;
    int vec;   // c takes four columns at once
};

template <typename T>
struct alignas(sizeof(T) * 4) Four {
    T e[4];
};

// Four adjacent columns of a row, ws their scales.
template <typename T>
__device__ __forceinline__ void epilogue4(const Args& g, int64_t row, int64_t col, i32x4 s, float as, const float (&ws)[4]) {
    if (row >= g.rows || col >= g.n) return;
    T* c = static_cast<T*>(g.c) + row * g.n + col;
    Four<T> y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y.e[i] = narrow<T>(static_cast<float>(s[i]) * (as * ws[i]));
    if (g.vec) {
        *reinterpret_cast<Four<T>*>(c) = y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < g.n) c[i] = y.e[i];
    }
}

// Tiles of 32 MB rows x 32 columns.  The four waves of a workgroup share the
// k range of its tile step by step, operands straight from global memory into
// registers (a wave's loads of a step are 1 KB each), and their sums meet in
// LDS.  Where the tiles are few, several workgroups share a tile's k range,
// store their sums in the workspace and the last one adds them (integers: the
// order does not matter).  16 x 2048 x 5632: 5.5 us (2.1 TB/s of weights; its
// waves wait for loads 81 % of their time, a step's after the other's); 4 x 8192 x
// 28672: 40 us (5.9 TB/s, repeated: part of the weights come from the last cache).
template <typename T, int MB>
__global__ __launch_bounds__(kT) void qmm_a8_kernel(const Args g) {
    __shared__ __align__(16) int sums[3][MB * 32 * 32];
    __shared__ unsigned ticket;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = static_cast<int>(blockIdx.x);
    const int split = id % g.splits;
    id /= g.splits;
    const int tile = id;
    const int tm = id % g.tiles_m, panel = id / g.tiles_m;
    // this wave's k steps
    const int ways = 4 * g.splits, way = 4 * split + wave;
    const int s0 = static_cast<int>(static_cast<int64_t>(g.steps) * way / ways);
    const int s1 = static_cast<int>(static_cast<int64_t>(g.steps) * (way + 1) / ways);
    const int8_t* wp = g.w + static_cast<int64_t>(panel) * g.steps * kBlockBytes + lane * 16;
    const int8_t* ap[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b)
        ap[b] = g.a + static_cast<int64_t>(min(tm * MB + b, g.row_blocks - 1)) * g.steps * kBlockBytes + lane * 16;
    // This thread's outputs: columns 4 (thread % 8) .., rows thread / 8 + 32 b.
    const int64_t row0 = static_cast<int64_t>(tm) * MB * 32 + threadIdx.x / 8;
    const int64_t col0 = static_cast<int64_t>(panel) * 32 + 4 * (threadIdx.x % 8);
    float as[MB], ws[4];
#pragma unroll
    for (int b = 0; b < MB; ++b) as[b] = g.a_scale[min(row0 + 32 * b, g.rows - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i) ws[i] = g.w_scale[min(col0 + i, g.n - 1)];
    i32x16 acc[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] = 0;
    for (int s = s0; s < s1; ++s) {
        const int64_t o = static_cast<int64_t>(s) * kBlockBytes;
        i32x4 wv[2], av[MB][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            wv[h] = *reinterpret_cast<const i32x4*>(wp + o + 1024 * h);
#pragma unroll
            for (int b = 0; b < MB; ++b) av[b][h] = *reinterpret_cast<const i32x4*>(ap[b] + o + 1024 * h);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int b = 0; b < MB; ++b) acc[b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[b][h], wv[h], acc[b], 0, 0, 0);
    }
    // Element e of lane l: row 8 (e / 4) + 4 (l / 32) + e % 4, column l % 32.
    if (wave > 0) {
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                sums[wave - 1][(b * 32 + 8 * (e / 4) + 4 * (lane / 32) + e % 4) * 32 + lane % 32] = acc[b][e];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int at = (b * 32 + 8 * (e / 4) + 4 * (lane / 32) + e % 4) * 32 + lane % 32;
                sums[0][at] += acc[b][e];
            }
    }
    __syncthreads();
    i32x4 mine[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        const int at = (b * kT + threadIdx.x) * 4;
        mine[b] = *reinterpret_cast<const i32x4*>(&sums[0][at]) + *reinterpret_cast<const i32x4*>(&sums[1][at]) +
                  *reinterpret_cast<const i32x4*>(&sums[2][at]);
    }
    constexpr uint32_t kPart = MB * 32 * 32 * 4;
    if (g.splits > 1) {
        char* tile_parts = reinterpret_cast<char*>(g.parts) + static_cast<int64_t>(tile) * g.splits * kPart;
        const __amdgpu_buffer_rsrc_t prs = buffer_rsrc(tile_parts, kPart * static_cast<uint32_t>(g.splits));
#pragma unroll
        for (int b = 0; b < MB; ++b)
            coherent_store16(prs, split * kPart + (b * kT + threadIdx.x) * 16, __builtin_bit_cast(u32x4, mine[b]));
        publish_partials();
        __syncthreads();
        if (threadIdx.x == 0) ticket = ticket_take(g.tickets + tile * kTicketStride, g.splits);
        __syncthreads();
        if (ticket != static_cast<unsigned>(g.splits - 1)) return;
        if (threadIdx.x == 0) __hip_atomic_store(g.tickets + tile * kTicketStride, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int s = 0; s < g.splits; ++s) {
            if (s == split) continue;
#pragma unroll
            for (int b = 0; b < MB; ++b)
                mine[b] += __builtin_bit_cast(i32x4, coherent_load16(prs, s * kPart + (b * kT + threadIdx.x) * 16));
        }
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) epilogue4<T>(g, row0 + 32 * b, col0, mine[b], as[b], ws);
}

// ---- Large products: tiles of BM x BN by 2 x WN waves, 64 k a stage.  The
// rows' blocks of a stage come in by 16-byte loads (WN blocks a load of the
// workgroup), wait in registers, kAhead stages early, and go to one of three
// LDS buffers as they are, so every LDS access is 1 KB of adjacent bytes; the
// columns' blocks go straight to the operand registers of the two waves that
// need them (through LDS as well: 570 us, 512 rows 19.6 us against 19.1).  A
// wave reads the rows of the next 32 k while it multiplies these, across stages
// too (the stage after next is being written meanwhile: the barrier at a
// stage's end orders both).  2048 x 8192 x 28672: 546 us, 1.76 POP/s (a large
// library product of 8-bit integers reaches 2.1 here): the matrix cores are
// busy 44 % of the cycles, the rest waits at the stages' barriers and for
// operands (512 x 2048 x 5632, tiles for two of three compute units: 16 us, 10 %);
// with both through LDS, 256 x 256 tiles with one wave a SIMD took 620, and 128 k a
// stage 725.
template <typename T, int BM, int BN, int WN>
__global__ __launch_bounds__(128 * WN, WN / 2) void qmm_a8_tile_kernel(const Args g) {
    constexpr int PA = BM / 32, PB = BN / 32;       // blocks of a stage
    constexpr int MT = BM / 64, NT = BN / WN / 32;  // a wave's 32 x 32 tiles
    constexpr int LA = PA / WN;                     // loads of a stage's rows, WN blocks each
    constexpr int kAhead = WN == 2 ? 3 : 4;
    constexpr int kStage = PA * kBlockBytes;
    __shared__ __align__(16) int8_t lds[3 * kStage];
    const int tiles_n = (g.panels + PB - 1) / PB, tiles_m = (g.row_blocks + PA - 1) / PA;
    // Workgroups go to the XCDs in turn: an XCD's are the row tiles of every
    // eighth column tile, which share that column's weights in its L2.
    const int xcd = static_cast<int>(blockIdx.x) % 8, j = static_cast<int>(blockIdx.x) / 8;
    // (scalars, which the buffer descriptors have to be made of)
    const int tm = __builtin_amdgcn_readfirstlane(j % tiles_m);
    const int tn = __builtin_amdgcn_readfirstlane(j / tiles_m * 8 + xcd);
    if (tn >= tiles_n) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave / WN, wc = wave % WN;

    // Blocks past the operands' ends, and stages past the last, read as zeros.
    const uint32_t pitch = static_cast<uint32_t>(g.steps) * kBlockBytes;
    const __amdgpu_buffer_rsrc_t ars = buffer_rsrc(g.a + static_cast<int64_t>(tm) * PA * pitch,
                                                   static_cast<uint32_t>(min(PA, g.row_blocks - tm * PA)) * pitch);
    const __amdgpu_buffer_rsrc_t brs = buffer_rsrc(g.w + static_cast<int64_t>(tn) * PB * pitch,
                                                   static_cast<uint32_t>(min(PB, g.panels - tn * PB)) * pitch);
    const uint32_t from = static_cast<uint32_t>(tid >> 7) * pitch + static_cast<uint32_t>(tid & 127) * 16;
    struct Rows {
        u32x4 v[LA];
    };
    struct Columns {
        i32x4 v[2][NT];
    };
    const auto at = [&](int stage) {
        return stage < g.steps ? static_cast<uint32_t>(stage) * kBlockBytes : 0x80000000u;
    };
    const auto load_rows = [&](int stage, Rows& t) {
        const uint32_t o = at(stage) + from;
#pragma unroll
        for (int u = 0; u < LA; ++u) t.v[u] = buffer_load16(ars, o + WN * u * pitch);
    };
    const uint32_t column = static_cast<uint32_t>(wc * NT) * pitch + lane * 16;
    const auto load_columns = [&](int stage, Columns& t) {
        const uint32_t o = at(stage) + column;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n)
                t.v[h][n] = __builtin_bit_cast(i32x4, buffer_load16(brs, o + n * pitch + 1024 * h));
    };
    const auto store = [&](const Rows& t, int8_t* to) {
#pragma unroll
        for (int u = 0; u < LA; ++u) *reinterpret_cast<u32x4*>(to + u * WN * kBlockBytes + tid * 16) = t.v[u];
    };
    i32x4 fa[2][MT];   // rows of this and the next 32 k
    const auto fetch = [&](const int8_t* stage, int h) {
        const int8_t* la = stage + wr * MT * kBlockBytes + h * 1024 + lane * 16;
#pragma unroll
        for (int i = 0; i < MT; ++i) fa[h][i] = *reinterpret_cast<const i32x4*>(la + i * kBlockBytes);
    };
    i32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][n][e] = 0;
    const auto multiply = [&](int h, const Columns& t) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
                acc[i][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[h][i], t.v[h][n], acc[i][n], 0, 0, 0);
    };

    Rows rows[kAhead];
    Columns columns[kAhead];
    {
        Rows t0, t1;
        load_rows(0, t0);
        load_rows(1, t1);
#pragma unroll
        for (int d = 0; d < kAhead; ++d) {
            load_columns(d, columns[d]);
            load_rows(2 + d, rows[d]);
        }
        store(t0, lds);
        store(t1, lds + kStage);
    }
    __syncthreads();
    int8_t *now = lds, *next = lds + kStage, *after = lds + 2 * kStage;
    fetch(now, 0);
    const auto advance = [&](int stage, Columns& c, Rows& t, bool more) {
        fetch(now, 1);
        multiply(0, c);
        store(t, after);   // stage + 2
        fetch(next, 0);
        multiply(1, c);
        if (more) {
            load_columns(stage + kAhead, c);
            load_rows(stage + 2 + kAhead, t);
        }
        __syncthreads();
        int8_t* first = now;
        now = next;
        next = after;
        after = first;
    };
    int stage = 0;
    for (; stage + kAhead <= g.steps; stage += kAhead) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d) advance(stage + d, columns[d], rows[d], true);
    }
#pragma unroll
    for (int d = 0; d < kAhead - 1; ++d)
        if (stage + d < g.steps) advance(stage + d, columns[d], rows[d], false);
    // Element e of lane l: row 8 (e / 4) + 4 (l / 32) + e % 4, column l % 32.
    // All the scales first: a load between two stores would wait for them.
    float as[MT][16], ws[NT];
    const int64_t row0 = (static_cast<int64_t>(tm) * PA + wr * MT) * 32 + 4 * (lane / 32);
    const int64_t col0 = (static_cast<int64_t>(tn) * PB + wc * NT) * 32 + lane % 32;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) as[i][e] = g.a_scale[min(row0 + 32 * i + 8 * (e / 4) + e % 4, g.rows - 1)];
#pragma unroll
    for (int n = 0; n < NT; ++n) ws[n] = g.w_scale[min(col0 + 32 * n, g.n - 1)];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int64_t row = row0 + 32 * i + 8 * (e / 4) + e % 4;
            T* c = static_cast<T*>(g.c) + row * g.n + col0;
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (row < g.rows && col0 + 32 * n < g.n)
                    c[32 * n] = narrow<T>(static_cast<float>(acc[i][n][e]) * (as[i][e] * ws[n]));
        }
}

struct Plan {
    int mb, splits;
    int wn;   // waves along n of the LDS kernel's 128 x 128 tiles; 0: the other kernel
    int64_t tiles_m, panels, bytes;
};

Plan plan(int64_t rows, int64_t k, int64_t n) {
    Plan p;
    const int64_t rb = blocks32(rows);
    // Large outputs: 128 x 128 tiles through LDS, with eight waves a tile where
    // there is not one for each compute unit.  With the staging, k = 2048, us with
    // eight waves, with four, without LDS: 300 x 5632 (132 tiles) 18.9, 20.4, 19.9;
    // 512 x 5632 (176) 20.7, 22.0, 22.3; 1000 x 2048 (128) 20.5, 22.1, 17.8; 2000 x
    // 2048 (256) 26.7, 27.1, 30.5; 700 x 5632 (264) 32.5, 28.4, 29.8; 1000 x 5632
    // (352) 34.9, 30.9, 35.1.
    const int64_t tiles = (rows + 127) / 128 * ((n + 127) / 128);
    p.wn = rows <= 128 || tiles < 160 ? 0 : tiles < 256 ? 4 : 2;
    p.mb = rb <= 1 ? 1 : rb <= 2 ? 2 : 4;
    p.tiles_m = (rb + p.mb - 1) / p.mb;
    p.panels = blocks32(n);
    const int64_t parts = p.tiles_m * p.panels;
    // Few tiles: workgroups that fill the GPU twice share the k, as long as a
    // wave keeps five steps (16 x 5632 x 2048: 10.5 us with four, 11.4 with eight,
    // 13.8 with one; 16 x 2048 x 5632: 8.6 with one, 9.3 with three; 32 x 8192 x
    // 8192: 17.7 with two, 19.6 with one; 16 x 2048 x 256, one workgroup for each
    // of eight panels: 8.3).
    int64_t s = parts < kMaxTiles ? kMaxTiles / parts : 1;
    s = std::max<int64_t>(std::min<int64_t>({s, kMaxSplits, steps64(k) / 20}), 1);
    p.splits = static_cast<int>(s);
    if (p.wn) {
        p.tiles_m = (rows + 127) / 128;
        p.splits = 1;
        p.bytes = 0;
        return p;
    }
    p.bytes = s > 1 ? kTicketBytes + parts * s * p.mb * 4096 : 0;
    return p;
}

int check_a8(int64_t rows, int64_t k, int64_t n, const char* who) {
    const std::string w(who);
    if (k < 1 || k > VM_HIP_A8_MAX_K) return fail_inval(w + ": k must be in [1, 131072]");
    if (rows < 0 || rows > VM_HIP_A8_MAX_ROWS || n < 0 || n > VM_HIP_A8_MAX_N)
        return fail_inval(w + ": rows or n out of range");
    if (blocks32(rows) * blocks32(n) > (1 << 27))   // (a launch has less than 2^32 threads)
        return fail_inval(w + ": too many outputs for one call");
    return 0;
}

bool known_dtype(int d) { return d == VM_HIP_DTYPE_F32 || d == VM_HIP_DTYPE_F16 || d == VM_HIP_DTYPE_BF16; }
bool off(const void* p, unsigned m) { return (reinterpret_cast<uintptr_t>(p) & m) != 0; }
unsigned element_mask(int d) { return d == VM_HIP_DTYPE_F32 ? 3 : 1; }

template <typename T>
int stage(const void* a, int64_t rows, int64_t k, void* staged, hipStream_t stream) {
    float* scales = reinterpret_cast<float*>(static_cast<char*>(staged) + staged_codes(rows, k));
    const bool spread = rows >= 256;
    const int64_t grid = spread ? (rows + 255) / 256 * 256 : rows;
    hipLaunchKernelGGL(a8_stage_row_kernel<T>, dim3(static_cast<unsigned>(grid)), dim3(kT), 0, stream,
                       static_cast<const T*>(a), static_cast<int8_t*>(staged), scales, rows, static_cast<int>(k),
                       static_cast<int>(steps64(k)), spread ? 1 : 0);
    return check_launch("a8_stage", stream);
}

template <typename T>
void launch(const Args& g, const Plan& p, hipStream_t stream) {
    const int mb = p.mb;
    if (p.wn) {
        const int64_t tiles_n = (g.n + 127) / 128;
        const dim3 d(static_cast<unsigned>(p.tiles_m * ((tiles_n + 7) / 8) * 8));
        if (p.wn == 4)
            hipLaunchKernelGGL((qmm_a8_tile_kernel<T, 128, 128, 4>), d, dim3(512), 0, stream, g);
        else
            hipLaunchKernelGGL((qmm_a8_tile_kernel<T, 128, 128, 2>), d, dim3(256), 0, stream, g);
        return;
    }
    const dim3 d(static_cast<unsigned>(p.tiles_m * p.panels * p.splits));
    if (mb == 1)
        hipLaunchKernelGGL((qmm_a8_kernel<T, 1>), d, dim3(kT), 0, stream, g);
    else if (mb == 2)
        hipLaunchKernelGGL((qmm_a8_kernel<T, 2>), d, dim3(kT), 0, stream, g);
    else
        hipLaunchKernelGGL((qmm_a8_kernel<T, 4>), d, dim3(kT), 0, stream, g);
}

}  // namespace
}  // namespace vmhip

using namespace vmhip;

extern "C" {

int64_t vm_hip_a8_weights_bytes(int64_t k, int64_t n) {
    clear_error();
    VM_TRY(check_a8(1, k, n, "a8_weights_bytes"));
    return blocks32(n) * steps64(k) * kBlockBytes;
}

int64_t vm_hip_a8_stage_bytes(int64_t rows, int64_t k) {
    clear_error();
    VM_TRY(check_a8(rows, k, 1, "a8_stage_bytes"));
    return staged_codes(rows, k) + blocks32(rows) * 32 * 4;
}

int64_t vm_hip_qmm_a8_workspace_bytes(int64_t rows, int64_t k, int64_t n) {
    clear_error();
    VM_TRY(check_a8(rows, k, n, "qmm_a8_workspace_bytes"));
    return rows && n ? plan(rows, k, n).bytes : 0;
}

int vm_hip_a8_pack(const int8_t* codes, int64_t k, int64_t n, void* packed, void* stream) {
    clear_error();
    VM_TRY(check_a8(1, k, n, "a8_pack"));
    if (n == 0) return 0;
    if (!codes || !packed) return fail_inval("a8_pack: null pointer");
    if (off(packed, 15)) return fail_inval("a8_pack: packed must be 16-byte aligned");
    const int64_t chunks = blocks32(n) * steps64(k) * (kBlockBytes / 16);
    const int64_t blocks = std::min<int64_t>((chunks + kT - 1) / kT, 65536);
    auto s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(a8_pack_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kT), 0, s, codes,
                       static_cast<int8_t*>(packed), k, n, steps64(k), chunks);
    return check_launch("a8_pack", s);
}

int vm_hip_a8_stage(const void* a, int dtype, int64_t rows, int64_t k, void* staged, void* stream) {
    clear_error();
    VM_TRY(check_a8(rows, k, 1, "a8_stage"));
    if (!known_dtype(dtype)) return fail_inval("a8_stage: dtype must be F32, F16 or BF16");
    if (rows == 0) return 0;
    if (!a || !staged) return fail_inval("a8_stage: null pointer");
    if (off(staged, 15) || off(a, element_mask(dtype))) return fail_inval("a8_stage: unaligned pointer");
    auto s = static_cast<hipStream_t>(stream);
    if (dtype == VM_HIP_DTYPE_F16) return stage<F16>(a, rows, k, staged, s);
    if (dtype == VM_HIP_DTYPE_BF16) return stage<BF16>(a, rows, k, staged, s);
    return stage<float>(a, rows, k, staged, s);
}

int vm_hip_qmm_a8(const void* staged, const void* packed, const float* scale, void* c, int c_dtype, int64_t rows,
                  int64_t k, int64_t n, void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    VM_TRY(check_a8(rows, k, n, "qmm_a8"));
    if (!known_dtype(c_dtype)) return fail_inval("qmm_a8: c_dtype must be F32, F16 or BF16");
    if (rows == 0 || n == 0) return 0;
    if (!staged || !packed || !scale || !c) return fail_inval("qmm_a8: null pointer");
    if (off(staged, 15) || off(packed, 15) || off(scale, 3) || off(c, element_mask(c_dtype)))
        return fail_inval("qmm_a8: unaligned pointer");
    const Plan p = plan(rows, k, n);
    if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || off(workspace, 15)))
        return fail_inval("qmm_a8: workspace smaller than vm_hip_qmm_a8_workspace_bytes or unaligned");
    Args g;
    g.a = static_cast<const int8_t*>(staged);
    g.a_scale = reinterpret_cast<const float*>(g.a + staged_codes(rows, k));
    g.w = static_cast<const int8_t*>(packed);
    g.w_scale = scale;
    g.c = c;
    g.tickets = static_cast<unsigned*>(workspace);
    g.parts = p.bytes > 0 ? reinterpret_cast<int*>(static_cast<char*>(workspace) + kTicketBytes) : nullptr;
    g.rows = rows;
    g.n = n;
    g.row_blocks = static_cast<int>(blocks32(rows));
    g.steps = static_cast<int>(steps64(k));
    g.panels = static_cast<int>(p.panels);
    g.tiles_m = static_cast<int>(p.tiles_m);
    g.splits = p.splits;
    const unsigned e = c_dtype == VM_HIP_DTYPE_F32 ? 4 : 2;
    g.vec = n % 4 == 0 && !off(c, 4 * e - 1);
    auto s = static_cast<hipStream_t>(stream);
    if (c_dtype == VM_HIP_DTYPE_F16)
        launch<F16>(g, p, s);
    else if (c_dtype == VM_HIP_DTYPE_BF16)
        launch<BF16>(g, p, s);
    else
        launch<float>(g, p, s);
    return check_launch("qmm_a8", s);
}

}  // extern "C"
