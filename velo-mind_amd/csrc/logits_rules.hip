// Penalties for repeated tokens, biases and grammar masks on logits, and the
// greedy token of what is left, in one pass.
//
// A workgroup takes a chunk of one row's vocabulary.  It requests its logits
// first; while they travel it counts, in LDS, how often each token of its
// chunk stands in the sequence's history and on the row's path (every
// workgroup of a row reads the whole history: a few KB from L2, against a
// counting pass and a vocabulary of counts in memory), and notes the last bias
// entry of each (integer maximum: the order of arrival does not matter).  Then
// each value is changed and stored, and the best one of the chunk goes to the
// workspace; the last workgroup of a row (atomic ticket) reduces the
// candidates, lowest index on ties.  Bound by HBM for large batches, by the
// chain of loads and the ticket for single rows.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "kv_q8.h"
#include "vm_device.h"
#include "vm_internal.h"

namespace vmhip {
namespace {

constexpr int kT = 256;
constexpr int kMaxRows = 65536;
constexpr int64_t kTicketBytes = kMaxRows * 4;

struct Args {
    vm_hip_logits_rules r;
    const void* logits;
    void* out;
    int32_t* tokens;
    const int32_t* counts;
    unsigned* tickets;
    float* best_value;     // [rows][chunks]
    int32_t* best_index;   // [rows][chunks]
    int64_t vocab;
    int rows, words, chunks, mask_words;
};

// Four adjacent logits, aligned as elements are; past `valid`: unspecified.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int valid, float (&x)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, int valid, float (&x)[4]) {
    if (valid >= 4) {
        __builtin_memcpy(x, p, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < valid ? p[i] : 0.0f;
    }
}
__device__ __forceinline__ void load4_bits(const uint16_t* p, int valid, uint16_t (&h)[4]) {
    if (valid >= 4) {
        __builtin_memcpy(h, p, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = i < valid ? p[i] : uint16_t(0);
    }
}
template <>
__device__ __forceinline__ void load4<F16>(const F16* p, int valid, float (&x)[4]) {
    uint16_t h[4];
    load4_bits(&p->bits, valid, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(__builtin_bit_cast(_Float16, h[i]));
}
template <>
__device__ __forceinline__ void load4<BF16>(const BF16* p, int valid, float (&x)[4]) {
    uint16_t h[4];
    load4_bits(&p->bits, valid, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(static_cast<uint32_t>(h[i]) << 16);
}

__device__ __forceinline__ void store4(float* p, int valid, const float (&x)[4]) {
    if (valid >= 4) {
        __builtin_memcpy(p, x, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = x[i];
    }
}
__device__ __forceinline__ void store4_bits(uint16_t* p, int valid, const uint16_t (&h)[4]) {
    if (valid >= 4) {
        __builtin_memcpy(p, h, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = h[i];
    }
}
__device__ __forceinline__ void store4(F16* p, int valid, const float (&x)[4]) {
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = narrow<F16>(x[i]).bits;
    store4_bits(&p->bits, valid, h);
}
__device__ __forceinline__ void store4(BF16* p, int valid, const float (&x)[4]) {
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = narrow<BF16>(x[i]).bits;
    store4_bits(&p->bits, valid, h);
}

// (v2, i2) beats (v1, i1); index -1: nothing.
__device__ __forceinline__ bool beats(float v1, int i1, float v2, int i2) {
    return i2 >= 0 && (i1 < 0 || v2 > v1 || (v2 == v1 && i2 < i1));
}

// The workgroup's best (every thread's candidate), in thread 0.
__device__ __forceinline__ void reduce_best(float& v, int& i, float* sv, int* si) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float ov = __shfl_xor(v, off, 64);
        const int oi = __shfl_xor(i, off, 64);
        if (beats(v, i, ov, oi)) v = ov, i = oi;
    }
    if ((threadIdx.x & 63) == 0) sv[threadIdx.x >> 6] = v, si[threadIdx.x >> 6] = i;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < kT / 64; ++w)
            if (beats(v, i, sv[w], si[w])) v = sv[w], i = si[w];
}

// Q groups of four values a thread: chunks of 1024 Q tokens.
template <typename T, int Q>
__global__ __launch_bounds__(kT) void logits_rules_kernel(const Args a) {
#pragma clang fp contract(off)
    constexpr int kChunk = 4 * kT * Q;
    __shared__ int seen[kChunk];    // occurrences of the chunk's tokens
    __shared__ int entry[kChunk];   // last bias entry + 1, 0: none
    __shared__ float sv[kT / 64];
    __shared__ int si[kT / 64];
    __shared__ unsigned ticket;
    const int chunk = static_cast<int>(blockIdx.x % a.chunks);
    const int64_t row = blockIdx.x / a.chunks;
    const int seq = static_cast<int>(row / a.rows), t = static_cast<int>(row - static_cast<int64_t>(seq) * a.rows);
    if (a.counts && t >= a.counts[seq]) return;
    const int64_t base = static_cast<int64_t>(chunk) * kChunk;
    const int size = static_cast<int>(min(a.vocab - base, static_cast<int64_t>(kChunk)));
    const int tid = threadIdx.x;
    const T* src = static_cast<const T*>(a.logits) + row * a.vocab + base;
    float x[Q][4];
    uint32_t allowed[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int o = 4 * (q * kT + tid);
        if (o < size) load4(src + o, size - o, x[q]);
        allowed[q] = 0xfu;
        if (a.r.allowed && o < size) allowed[q] = a.r.allowed[row * a.mask_words + (base + o) / 32] >> (o & 31);
    }
    const bool counting = (a.r.history || a.r.drafted) && (a.r.repetition || a.r.frequency || a.r.presence);
    const bool biased = a.r.bias_tokens != nullptr;
    if (counting || biased) {
        for (int i = tid; i < kChunk; i += kT) seen[i] = 0, entry[i] = 0;
        __syncthreads();
        if (counting) {
            const auto count = [&](int token) {
                const int64_t at = static_cast<int64_t>(token) - base;
                if (at >= 0 && at < size) atomicAdd(&seen[at], 1);
            };
            if (a.r.history) {
                const int32_t* h = a.r.history + seq * a.r.history_stride;
                const int64_t n = min(max(static_cast<int64_t>(a.r.history_lengths[seq]), int64_t(0)), a.r.history_stride);
                for (int64_t i = tid; i < n; i += kT) count(h[i]);
            }
            if (a.r.drafted) {
                const int32_t* d = a.r.drafted + static_cast<int64_t>(seq) * a.rows;
                for (int j = tid; j < a.rows; j += kT)
                    if (a.r.tree ? a.r.tree[row * a.words + j / 64] >> (j & 63) & 1 : j <= t) count(d[j]);
            }
        }
        if (biased) {
            const int32_t* b = a.r.bias_tokens + seq * a.r.bias_stride;
            const int64_t n = min(max(static_cast<int64_t>(a.r.bias_lengths[seq]), int64_t(0)), a.r.bias_stride);
            for (int64_t i = tid; i < n; i += kT) {
                const int64_t at = static_cast<int64_t>(b[i]) - base;
                if (at >= 0 && at < size) atomicMax(&entry[at], static_cast<int>(i) + 1);
            }
        }
        __syncthreads();
        const float rep = a.r.repetition ? a.r.repetition[seq] : 1.0f;
        const float freq = a.r.frequency ? a.r.frequency[seq] : 0.0f;
        const float pres = a.r.presence ? a.r.presence[seq] : 0.0f;
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int o = 4 * (q * kT + tid) + e;
                const int n = seen[o];
                if (n > 0) {
                    float v = x[q][e];
                    if (a.r.repetition) v = v > 0.0f ? v / rep : v * rep;
                    if (a.r.frequency) v = v - static_cast<float>(n) * freq;
                    if (a.r.presence) v = v - pres;
                    x[q][e] = v;
                }
                if (entry[o] > 0) x[q][e] = x[q][e] + a.r.bias_values[seq * a.r.bias_stride + entry[o] - 1];
            }
    }
    float best = -INFINITY;
    int index = -1;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int o = 4 * (q * kT + tid);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!(allowed[q] >> e & 1)) x[q][e] = -INFINITY;
            if (o + e < size && x[q][e] > best) best = x[q][e], index = static_cast<int>(base) + o + e;
        }
        if (a.out && o < size) store4(static_cast<T*>(a.out) + row * a.vocab + base + o, size - o, x[q]);
    }
    if (!a.tokens) return;
    reduce_best(best, index, sv, si);
    if (a.chunks > 1) {
        if (tid == 0) {
            coherent_store(a.best_value + row * a.chunks + chunk, best);
            __hip_atomic_store(a.best_index + row * a.chunks + chunk, index, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            publish_partials();
            ticket = ticket_take(a.tickets + row, a.chunks);
        }
        __syncthreads();
        if (ticket != static_cast<unsigned>(a.chunks - 1)) return;
        best = -INFINITY;
        index = -1;
        for (int c = tid; c < a.chunks; c += kT) {
            const float v = coherent_load(a.best_value + row * a.chunks + c);
            const int i = __hip_atomic_load(a.best_index + row * a.chunks + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (beats(best, index, v, i)) best = v, index = i;
        }
        __syncthreads();   // sv and si are reused
        reduce_best(best, index, sv, si);
    }
    if (tid == 0) {
        a.tokens[row] = index;
        if (a.chunks > 1) __hip_atomic_store(a.tickets + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

// Tokens of a workgroup: 1024 while 4096 would leave the GPU idle.
int chunk_of(int64_t rows, int64_t vocab) { return rows * ((vocab + 4095) / 4096) >= 512 ? 4096 : 1024; }

int check_shape(int64_t seqs, int64_t rows, int64_t vocab) {
    if (seqs < 0 || rows < 0 || seqs > kMaxRows || rows > kMaxRows || seqs * rows > kMaxRows)
        return fail_inval("logits_rules: seqs * rows must be in [0, 65536]");
    if (vocab < 1 || vocab > 0x7fffffff) return fail_inval("logits_rules: vocab must be in [1, 2^31)");
    if (seqs * rows * ((vocab + 1023) / 1024) > 0x7fffffff) return fail_inval("logits_rules: too many values for one call");
    return 0;
}

int64_t candidates(int64_t rows, int64_t vocab) {
    const int64_t c = chunk_of(rows, vocab);
    return rows * ((vocab + c - 1) / c);
}

template <typename T>
void launch(const Args& a, int chunk, int64_t grid, hipStream_t stream) {
    if (chunk == 4096)
        hipLaunchKernelGGL((logits_rules_kernel<T, 4>), dim3(static_cast<unsigned>(grid)), dim3(kT), 0, stream, a);
    else
        hipLaunchKernelGGL((logits_rules_kernel<T, 1>), dim3(static_cast<unsigned>(grid)), dim3(kT), 0, stream, a);
}

}  // namespace
}  // namespace vmhip

using namespace vmhip;

extern "C" {

int64_t vm_hip_logits_rules_workspace_bytes(int64_t seqs, int64_t rows, int64_t vocab) {
    clear_error();
    VM_TRY(check_shape(seqs, rows, vocab));
    return seqs * rows ? kTicketBytes + candidates(seqs * rows, vocab) * 8 : 0;
}

int vm_hip_logits_rules_apply(const vm_hip_logits_rules* rules, const void* logits, void* out, int dtype,
                              int32_t* tokens, int64_t seqs, int64_t rows, int64_t vocab, const int32_t* counts,
                              void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    VM_TRY(check_shape(seqs, rows, vocab));
    if (!rules) return fail_inval("logits_rules: null rules");
    if (dtype != VM_HIP_DTYPE_F32 && dtype != VM_HIP_DTYPE_F16 && dtype != VM_HIP_DTYPE_BF16)
        return fail_inval("logits_rules: dtype must be F32, F16 or BF16");
    if (rules->history && (!rules->history_lengths || rules->history_stride < 0))
        return fail_inval("logits_rules: history needs its lengths and stride");
    if (rules->bias_tokens &&
        (!rules->bias_values || !rules->bias_lengths || rules->bias_stride < 0 || rules->bias_stride > 0x7ffffffe))
        return fail_inval("logits_rules: bias_tokens need their values, lengths and stride");
    if (seqs * rows == 0) return 0;
    if (!logits || (!out && !tokens)) return fail_inval("logits_rules: null pointer");
    const unsigned m = dtype == VM_HIP_DTYPE_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & m)
        return fail_inval("logits_rules: logits or out not aligned to its elements");
    if (tokens && (!workspace || workspace_bytes < vm_hip_logits_rules_workspace_bytes(seqs, rows, vocab) ||
                   (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))
        return fail_inval("logits_rules: workspace smaller than vm_hip_logits_rules_workspace_bytes or unaligned");
    Args a;
    a.r = *rules;
    a.logits = logits;
    a.out = out;
    a.tokens = tokens;
    a.counts = counts;
    const int64_t n = candidates(seqs * rows, vocab);
    a.tickets = static_cast<unsigned*>(workspace);
    a.best_value = tokens ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kTicketBytes) : nullptr;
    a.best_index = tokens ? reinterpret_cast<int32_t*>(a.best_value + n) : nullptr;
    a.vocab = vocab;
    a.rows = static_cast<int>(rows);
    a.words = static_cast<int>((rows + 63) / 64);
    a.mask_words = static_cast<int>((vocab + 31) / 32);
    const int chunk = chunk_of(seqs * rows, vocab);
    a.chunks = static_cast<int>((vocab + chunk - 1) / chunk);
    auto s = static_cast<hipStream_t>(stream);
    if (dtype == VM_HIP_DTYPE_F16)
        launch<F16>(a, chunk, n, s);
    else if (dtype == VM_HIP_DTYPE_BF16)
        launch<BF16>(a, chunk, n, s);
    else
        launch<float>(a, chunk, n, s);
    return check_launch("logits_rules", s);
}

}  // extern "C"
