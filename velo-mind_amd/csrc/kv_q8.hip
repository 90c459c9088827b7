// The INT8 KV cache: rotation and quantization of a projection's keys and
// values as they are written, the cache read back as numbers, and the rows of
// a tree's accepted path moved together.
//
// Quantization (quant.cpp:74-104 per token and head instead of per column):
// s = max|x| / 127, c = round(x * (1 / s)) half away from zero, clamped; the
// division and reciprocal are correctly rounded (build flags) and nothing is
// contracted, so codes and scales are the same bits wherever the formula is
// evaluated in fp32.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "kv_q8.h"
#include "vm_device.h"
#include "vm_internal.h"

namespace vmhip {

int check_kv_q8(const vm_hip_kv_q8* c, const char* who) {
    const std::string w(who);
    if (!c) return fail_inval(w + ": null cache");
    if (c->head_dim != 64 && c->head_dim != 128) return fail_inval(w + ": head_dim must be 64 or 128");
    if (c->batch < 0 || c->batch > 65535 || c->kv_heads < 1 || c->kv_heads > 4096 || c->max_seq < 1 ||
        c->max_seq > 0x7fffffff / c->head_dim)
        return fail_inval(w + ": batch, kv_heads or max_seq out of range");
    if (c->batch == 0) return 0;
    if (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales) return fail_inval(w + ": null cache pointer");
    const auto off = [](const void* p, unsigned m) { return (reinterpret_cast<uintptr_t>(p) & m) != 0; };
    if (off(c->k_codes, 15) || off(c->v_codes, 15)) return fail_inval(w + ": codes must be 16-byte aligned");
    if (off(c->k_scales, 3) || off(c->v_scales, 3)) return fail_inval(w + ": scales must be 4-byte aligned");
    return 0;
}

namespace {

constexpr int kT = 256;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool known_dtype(int d) { return d == VM_HIP_DTYPE_F32 || d == VM_HIP_DTYPE_F16 || d == VM_HIP_DTYPE_BF16; }

// N adjacent values of a row.
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T e[N];
};

// ---- Append.  Sixteen lanes own one head row of one token: lane i holds
// elements i D / 32 .. of the lower half and the same of the upper half, the
// pairs that a rotation combines, so the row's maximum is four DPP steps away
// and nothing touches LDS.  Bound: one read of qkv, one write of q, codes and
// scales; small calls wait for the chain pos -> table -> store (one token of 40
// heads of 64: 2.6 us; 128 tokens of 80 heads of 128, bf16: 5.2; a prompt of 2000
// such tokens: 18, 4.3 TB/s).
template <typename T, int D>
__global__ __launch_bounds__(kT) void kv_q8_append_kernel(const vm_hip_kv_q8 c, const T* __restrict__ qkv,
                                                          const float* __restrict__ cos_t,
                                                          const float* __restrict__ sin_t,
                                                          const int32_t* __restrict__ pos,
                                                          const int32_t* __restrict__ counts,
                                                          const int32_t* __restrict__ depths, T* __restrict__ q_out,
                                                          int rows, int heads, int64_t total) {
#pragma clang fp contract(off)
    constexpr int N = D / 32;   // pairs of a lane
    const int hk = static_cast<int>(c.kv_heads);
    const int all = heads + 2 * hk;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (kT / 16) + threadIdx.x / 16;
    if (item >= total) return;   // whole 16-lane groups leave
    const int i = threadIdx.x & 15;
    const int64_t token = item / all;
    const int h = static_cast<int>(item - token * all);
    const int b = static_cast<int>(token / rows), t = static_cast<int>(token - static_cast<int64_t>(b) * rows);
    const int64_t p0 = pos[b];
    const int64_t p = p0 + t;
    if (p < 0 || p >= c.max_seq || (counts && t >= counts[b])) return;
    const T* src = qkv + (token * all + h) * D + i * N;
    const Vec<T, N> xl = *reinterpret_cast<const Vec<T, N>*>(src);
    const Vec<T, N> xh = *reinterpret_cast<const Vec<T, N>*>(src + D / 2);
    float lo[N], hi[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        lo[e] = widen(xl.e[e]);
        hi[e] = widen(xh.e[e]);
    }
    if (h < heads + hk) {
        int64_t turn = p0 + (depths ? depths[token] : t);
        turn = turn < 0 ? 0 : turn < c.max_seq ? turn : c.max_seq - 1;
        const float* cp = cos_t + turn * (D / 2) + i * N;
        const float* sp = sin_t + turn * (D / 2) + i * N;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float cs = cp[e], sn = sp[e];
            const float a = lo[e], bb = hi[e];
            lo[e] = a * cs - bb * sn;
            hi[e] = bb * cs + a * sn;
        }
    }
    if (h < heads) {
        Vec<T, N> yl, yh;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            yl.e[e] = narrow<T>(lo[e]);
            yh.e[e] = narrow<T>(hi[e]);
        }
        T* q = q_out + ((static_cast<int64_t>(b) * heads + h) * rows + t) * D + i * N;
        *reinterpret_cast<Vec<T, N>*>(q) = yl;
        *reinterpret_cast<Vec<T, N>*>(q + D / 2) = yh;
        return;
    }
    // Magnitudes compare as integers, and infinities and NaN stay on top.
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        m = max(m, __float_as_uint(lo[e]) & 0x7fffffffu);
        m = max(m, __float_as_uint(hi[e]) & 0x7fffffffu);
    }
#pragma unroll
    for (int s = 1; s < 16; s <<= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), s, 64)));
    const Q8Scale q8 = q8_scale(m);
    const bool value = h >= heads + hk;
    const int kh = h - heads - (value ? hk : 0);
    const int64_t row = (static_cast<int64_t>(b) * hk + kh) * c.max_seq + p;
    int8_t* codes = (value ? c.v_codes : c.k_codes) + row * D + i * N;
    Vec<int8_t, N> cl, ch;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        cl.e[e] = q8_code(lo[e], q8.inv);
        ch.e[e] = q8_code(hi[e], q8.inv);
    }
    *reinterpret_cast<Vec<int8_t, N>*>(codes) = cl;
    *reinterpret_cast<Vec<int8_t, N>*>(codes + D / 2) = ch;
    if (i == 0) (value ? c.v_scales : c.k_scales)[row] = q8.scale;
}

// ---- Read back: four codes of a row per thread and step, so that a wave
// writes 1 KB of adjacent fp32 values.  Bound by HBM (five bytes per code): 8
// sequences x 4000 tokens x 8 heads of 128, K and V, 62 us, 5.4 TB/s.
template <typename T>
__global__ __launch_bounds__(kT) void kv_q8_read_kernel(const vm_hip_kv_q8 c, T* __restrict__ k_out,
                                                        T* __restrict__ v_out, int64_t first, int64_t rows,
                                                        int64_t quads) {
    const bool value = blockIdx.y != 0 || !k_out;
    const int8_t* codes = value ? c.v_codes : c.k_codes;
    const float* scales = value ? c.v_scales : c.k_scales;
    T* out = value ? v_out : k_out;
    const int shift = c.head_dim == 64 ? 4 : 5;   // quads of a row
    const int64_t step = static_cast<int64_t>(gridDim.x) * kT;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * kT + threadIdx.x; u < quads; u += step) {
        const int64_t r = u >> shift;             // output row: (sequence, head, token)
        const int64_t head = r / rows;
        const int64_t row = head * c.max_seq + first + (r - head * rows);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + (row << (shift + 2)) +
                                                              ((u & ((1 << shift) - 1)) << 2));
        const float s = scales[row];
        Vec<T, 4> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.e[e] = narrow<T>(static_cast<float>(static_cast<int8_t>(w >> (8 * e))) * s);
        *reinterpret_cast<Vec<T, 4>*>(out + 4 * u) = y;
    }
}

// ---- Keep: one workgroup per (sequence, head, keys | values) holds every
// kept row in registers (at most 256 rows: eight 16-byte pieces a thread)
// before the first store, so sources and targets may overlap in any way.  8
// rows of 8 sequences x 8 heads of 128: 2.8-3.6 us, a launch and a round trip.
constexpr int kKeepPieces = VM_HIP_KV_Q8_KEEP_MAX * 128 / 16 / kT;

__global__ __launch_bounds__(kT) void kv_q8_keep_kernel(const vm_hip_kv_q8 c, const int32_t* __restrict__ pos,
                                                        const int32_t* __restrict__ kept,
                                                        const int32_t* __restrict__ kept_counts, int width) {
    const int64_t head = blockIdx.x;
    const int b = static_cast<int>(head / c.kv_heads);
    int8_t* codes = blockIdx.y ? c.v_codes : c.k_codes;
    float* scales = blockIdx.y ? c.v_scales : c.k_scales;
    const int n = min(max(kept_counts[b], 0), width);
    const int64_t p0 = pos[b];
    const int32_t* from = kept + static_cast<int64_t>(b) * width;
    const int per_row = static_cast<int>(c.head_dim / 16);
    const int64_t base = head * c.max_seq;
    const auto source = [&](int i) -> int64_t {   // the row that entry i moves, -1: skipped
        const int64_t s = p0 + from[i], d = p0 + i;
        return s < 0 || s >= c.max_seq || d < 0 || d >= c.max_seq ? -1 : s;
    };
    u32x4 piece[kKeepPieces];
    bool moves[kKeepPieces];
#pragma unroll
    for (int u = 0; u < kKeepPieces; ++u) {
        const int e = u * kT + threadIdx.x, i = e / per_row;
        const int64_t s = i < n ? source(i) : -1;
        moves[u] = s >= 0;
        if (moves[u])
            piece[u] = *reinterpret_cast<const u32x4*>(codes + (base + s) * c.head_dim + (e % per_row) * 16);
    }
    const int64_t s1 = static_cast<int>(threadIdx.x) < n ? source(threadIdx.x) : -1;
    const float sc = s1 >= 0 ? scales[base + s1] : 0.0f;
    publish_partials();   // this thread's loads have arrived
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kKeepPieces; ++u) {
        const int e = u * kT + threadIdx.x, i = e / per_row;
        if (moves[u])
            *reinterpret_cast<u32x4*>(codes + (base + p0 + i) * c.head_dim + (e % per_row) * 16) = piece[u];
    }
    if (s1 >= 0) scales[base + p0 + threadIdx.x] = sc;
}

template <typename T>
int append(const vm_hip_kv_q8& c, const void* qkv, int64_t rows, int64_t heads, const float* cos_t, const float* sin_t,
           const int32_t* pos, const int32_t* counts, const int32_t* depths, void* q_out, int64_t total,
           hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((total + kT / 16 - 1) / (kT / 16)));
    if (c.head_dim == 64)
        hipLaunchKernelGGL((kv_q8_append_kernel<T, 64>), grid, dim3(kT), 0, stream, c, static_cast<const T*>(qkv), cos_t,
                           sin_t, pos, counts, depths, static_cast<T*>(q_out), static_cast<int>(rows),
                           static_cast<int>(heads), total);
    else
        hipLaunchKernelGGL((kv_q8_append_kernel<T, 128>), grid, dim3(kT), 0, stream, c, static_cast<const T*>(qkv), cos_t,
                           sin_t, pos, counts, depths, static_cast<T*>(q_out), static_cast<int>(rows),
                           static_cast<int>(heads), total);
    return check_launch("kv_q8_append", stream);
}

template <typename T>
int read(const vm_hip_kv_q8& c, int64_t first, int64_t rows, void* k_out, void* v_out, hipStream_t stream) {
    const int64_t quads = c.batch * c.kv_heads * rows * (c.head_dim / 4);
    const int64_t blocks = (quads + kT - 1) / kT;
    const dim3 grid(static_cast<unsigned>(blocks < 16384 ? blocks : 16384), k_out && v_out ? 2 : 1);
    hipLaunchKernelGGL(kv_q8_read_kernel<T>, grid, dim3(kT), 0, stream, c, static_cast<T*>(k_out),
                       static_cast<T*>(v_out), first, rows, quads);
    return check_launch("kv_q8_read", stream);
}

}  // namespace
}  // namespace vmhip

using namespace vmhip;

extern "C" {

int vm_hip_kv_q8_append(const vm_hip_kv_q8* cache, const void* qkv, int dtype, int64_t rows, int64_t heads,
                        const float* cos_table, const float* sin_table, const int32_t* pos, const int32_t* counts,
                        const int32_t* depths, void* q_out, void* stream) {
    clear_error();
    VM_TRY(check_kv_q8(cache, "kv_q8_append"));
    if (!known_dtype(dtype)) return fail_inval("kv_q8_append: dtype must be F32, F16 or BF16");
    if (rows < 0 || rows > (1 << 20) || heads < 1 || heads > 65536 || heads % cache->kv_heads)
        return fail_inval("kv_q8_append: bad rows or heads");
    if (rows == 0 || cache->batch == 0) return 0;
    if (!qkv || !cos_table || !sin_table || !pos || !q_out) return fail_inval("kv_q8_append: null pointer");
    if (!aligned16(qkv) || !aligned16(q_out)) return fail_inval("kv_q8_append: qkv and q_out must be 16-byte aligned");
    const int64_t total = cache->batch * rows * (heads + 2 * cache->kv_heads);
    if (total >= (1 << 28))   // (a launch has less than 2^32 threads)
        return fail_inval("kv_q8_append: too many tokens for one call");
    auto s = static_cast<hipStream_t>(stream);
    if (dtype == VM_HIP_DTYPE_F16)
        return append<F16>(*cache, qkv, rows, heads, cos_table, sin_table, pos, counts, depths, q_out, total, s);
    if (dtype == VM_HIP_DTYPE_BF16)
        return append<BF16>(*cache, qkv, rows, heads, cos_table, sin_table, pos, counts, depths, q_out, total, s);
    return append<float>(*cache, qkv, rows, heads, cos_table, sin_table, pos, counts, depths, q_out, total, s);
}

int vm_hip_kv_q8_read(const vm_hip_kv_q8* cache, int64_t first, int64_t rows, void* k_out, void* v_out, int dtype,
                      void* stream) {
    clear_error();
    VM_TRY(check_kv_q8(cache, "kv_q8_read"));
    if (!known_dtype(dtype)) return fail_inval("kv_q8_read: dtype must be F32, F16 or BF16");
    if (first < 0 || rows < 0 || first > cache->max_seq || rows > cache->max_seq - first)
        return fail_inval("kv_q8_read: rows outside the cache");
    if (rows == 0 || cache->batch == 0) return 0;
    if (!k_out && !v_out) return fail_inval("kv_q8_read: null pointer");
    if (!aligned16(k_out) || !aligned16(v_out)) return fail_inval("kv_q8_read: outputs must be 16-byte aligned");
    auto s = static_cast<hipStream_t>(stream);
    if (dtype == VM_HIP_DTYPE_F16) return read<F16>(*cache, first, rows, k_out, v_out, s);
    if (dtype == VM_HIP_DTYPE_BF16) return read<BF16>(*cache, first, rows, k_out, v_out, s);
    return read<float>(*cache, first, rows, k_out, v_out, s);
}

int vm_hip_kv_q8_keep(const vm_hip_kv_q8* cache, const int32_t* pos, const int32_t* kept, const int32_t* kept_counts,
                      int64_t width, void* stream) {
    clear_error();
    VM_TRY(check_kv_q8(cache, "kv_q8_keep"));
    if (width < 0 || width > VM_HIP_KV_Q8_KEEP_MAX) return fail_inval("kv_q8_keep: width must be in [0, 256]");
    if (cache->batch * cache->kv_heads >= (1 << 24)) return fail_inval("kv_q8_keep: too many heads for one call");
    if (width == 0 || cache->batch == 0) return 0;
    if (!pos || !kept || !kept_counts) return fail_inval("kv_q8_keep: null pointer");
    auto s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(cache->batch * cache->kv_heads), 2);
    hipLaunchKernelGGL(kv_q8_keep_kernel, grid, dim3(kT), 0, s, *cache, pos, kept, kept_counts,
                       static_cast<int>(width));
    return check_launch("kv_q8_keep", s);
}

}  // extern "C"
