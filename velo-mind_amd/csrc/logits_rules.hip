// Penalties for repeated tokens, biases and grammar masks on logits, and the
// greedy token of what is left, in one pass.
//
// A workgroup takes up to four rows of one sequence and a range of the
// vocabulary, 1024 tokens (four a thread) at a time.  For each such chunk it
// counts in LDS how often its tokens stand in the history, which its threads
// keep in registers (up to 2048 tokens; every workgroup of a sequence reads
// the whole history: a few KB from L2, against a counting pass and a
// vocabulary of counts in memory), notes the last bias entry of each (integer
// maximum: the order of arrival does not matter) and counts the nodes on each
// row's path; the next chunk's logits are on their way meanwhile.  Every
// thread keeps its best value of each row; at the end the workgroup's best go
// to the workspace, and the last workgroup of a row (atomic ticket) reduces
// the candidates, lowest index on ties.  64 x 128256 fp32 behind 6000 tokens of
// history: 25 us, 2.6 TB/s (waves wait 60 % of their time, VALU instructions are 10
// us of it; with twice the history in registers three workgroups fit a compute
// unit instead of four: 29.2); 1 x 32000: 6.6 us (the chain lists - LDS - biases -
// ticket).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "kv_q8.h"
#include "vm_device.h"
#include "vm_internal.h"

namespace vmhip {
namespace {

constexpr int kT = 256;
constexpr int kMaxRows = 65536;
constexpr int64_t kMaxList = 1 << 30;   // entries of a history or a bias list
// A row's ticket has a 64-byte line of its own: tickets of 64 rows in two lines
// took the 8064 workgroups of 64 x 128256 logits 14 us of 37.
constexpr int kTicketStride = 16;

constexpr int kChunk = 4 * kT;        // tokens that a workgroup holds at a time
constexpr int kRowBatch = 4;          // rows of a workgroup
constexpr int kTargetGroups = 1024;    // workgroups that are resident together

struct Args {
    vm_hip_logits_rules r;
    const void* logits;
    void* out;
    int32_t* tokens;
    const int32_t* counts;
    unsigned* tickets;
    uint64_t* candidates;   // [rows][ranges]
    int64_t vocab;
    int rows, words, chunks, mask_words, groups, ranges;
};

// Four adjacent logits, aligned as elements are; past `valid`: unspecified.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int valid, float (&x)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, int valid, float (&x)[4]) {
    if (valid >= 4) {
        __builtin_memcpy(x, p, 16);
    } else {
        p = apart(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < valid ? p[i] : 0.0f;
    }
}
__device__ __forceinline__ void load4_bits(const uint16_t* p, int valid, uint16_t (&h)[4]) {
    if (valid >= 4) {
        __builtin_memcpy(h, p, 8);
    } else {
        p = apart(p);
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
        p = apart(p);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = x[i];
    }
}
__device__ __forceinline__ void store4_bits(uint16_t* p, int valid, const uint16_t (&h)[4]) {
    if (valid >= 4) {
        __builtin_memcpy(p, h, 8);
    } else {
        p = apart(p);
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

// A value and its token as one number that compares as "larger, or equal and
// of a lower token"; 0: none.
__device__ __forceinline__ uint64_t candidate(float v, int token) {
    if (token < 0) return 0;
    const uint32_t bits = __float_as_uint(v + 0.0f);   // (-0 equals 0)
    const uint32_t order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return static_cast<uint64_t>(order) << 32 | ~static_cast<uint32_t>(token);
}
__device__ __forceinline__ int candidate_token(uint64_t k) { return k ? static_cast<int>(~static_cast<uint32_t>(k)) : -1; }

// The wave's best of N rows, in every lane.
template <int N>
__device__ __forceinline__ void wave_best(uint64_t (&k)[N]) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        uint64_t o[N];
#pragma unroll
        for (int b = 0; b < N; ++b)
            o[b] = static_cast<uint64_t>(static_cast<uint32_t>(__shfl_xor(static_cast<int>(k[b] >> 32), off, 64))) << 32 |
                   static_cast<uint32_t>(__shfl_xor(static_cast<int>(k[b]), off, 64));
#pragma unroll
        for (int b = 0; b < N; ++b) k[b] = max(k[b], o[b]);
    }
}

template <typename T, int RB>
__global__ __launch_bounds__(kT, 4) void logits_rules_kernel(const Args a) {
#pragma clang fp contract(off)
    __shared__ __align__(16) int seen_lds[kChunk];        // occurrences in the history
    __shared__ __align__(16) int entry_lds[kChunk];       // last bias entry + 1, 0: none
    __shared__ __align__(16) int path_lds[RB][kChunk];    // occurrences on a row's path
    __shared__ uint64_t wave_key[RB][kT / 64];
    int id = static_cast<int>(blockIdx.x);
    const int range = id % a.ranges;
    id /= a.ranges;
    const int t0 = id % a.groups * RB, seq = id / a.groups;
    const int nodes = a.counts ? min(a.counts[seq], a.rows) : a.rows;   // the others are padding
    const int n_rows = min(nodes - t0, RB);
    if (n_rows <= 0) return;
    const int c0 = static_cast<int>(static_cast<int64_t>(a.chunks) * range / a.ranges);
    const int c1 = static_cast<int>(static_cast<int64_t>(a.chunks) * (range + 1) / a.ranges);
    const int tid = threadIdx.x, mine = 4 * tid;
    const int64_t row0 = static_cast<int64_t>(seq) * a.rows + t0;

    const bool penalties = a.r.repetition || a.r.frequency || a.r.presence;
    const bool histories = a.r.history && penalties, paths = a.r.drafted && penalties;
    // The lists, by their strides: the lengths are still on their way.
    constexpr int kVec = 2;
    const int stride = histories ? static_cast<int>(a.r.history_stride) : 0;
    const int32_t* history = a.r.history + seq * a.r.history_stride;
    int32_t h[kVec][4];
    const auto load_history = [&](int begin) {
#pragma unroll
        for (int u = 0; u < kVec; ++u) {
            const int i = begin + u * kChunk + mine;
            if (i + 4 <= stride) {
                __builtin_memcpy(h[u], history + i, 16);
            } else {
                const int32_t* p = apart(history);
#pragma unroll
                for (int e = 0; e < 4; ++e) h[u][e] = i + e < stride ? p[i + e] : -1;
            }
        }
    };
    if (stride) load_history(0);
    const int bias_stride = a.r.bias_tokens ? static_cast<int>(a.r.bias_stride) : 0;
    const int32_t* bias_tokens = a.r.bias_tokens + seq * a.r.bias_stride;
    const int first_bias = tid < bias_stride ? bias_tokens[tid] : -1;
    // A thread's (row, node) pairs: the node's token if it lies on the row's
    // path, else one that matches nothing.
    const int pairs = paths ? n_rows * nodes : 0;
    const auto path_token = [&](int pair) {
        const int r = pair / nodes, j = pair - r * nodes;
        const int token = a.r.drafted[row0 - t0 + j];
        const uint64_t on = a.r.tree ? a.r.tree[(row0 + r) * a.words + j / 64] >> (j & 63) & 1 : j <= t0 + r;
        return on ? token : -1;
    };
    const int first_path = tid < pairs ? path_token(tid) : -1;

    float x[RB][4];
    uint32_t allowed[RB];
    const auto load_rows = [&](int chunk) {
        const int64_t base = static_cast<int64_t>(chunk) * kChunk;
        const int valid = static_cast<int>(min(a.vocab - base, static_cast<int64_t>(kChunk))) - mine;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            allowed[b] = 0xfu;
            if (b < n_rows && valid > 0) {
                const T* from = static_cast<const T*>(a.logits) + (row0 + b) * a.vocab + base;   // (of the whole wave)
                load4(from + mine, valid, x[b]);
                if (a.r.allowed) {
                    const uint32_t* words = a.r.allowed + (row0 + b) * a.mask_words + base / 32;
                    allowed[b] = words[mine / 32] >> (mine & 31);
                }
            }
        }
    };
    if (c0 < c1) load_rows(c0);
    const int history_n = histories ? min(max(a.r.history_lengths[seq], 0), stride) : 0;
    const auto cut_history = [&](int begin) {   // past the length: what matches nothing
#pragma unroll
        for (int u = 0; u < kVec; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (begin + u * kChunk + mine + e >= history_n) h[u][e] = -1;
    };
    cut_history(0);
    const int bias_n = bias_stride ? min(max(a.r.bias_lengths[seq], 0), bias_stride) : 0;
    const float rep = a.r.repetition ? a.r.repetition[seq] : 1.0f;
    const float freq = a.r.frequency ? a.r.frequency[seq] : 0.0f;
    const float pres = a.r.presence ? a.r.presence[seq] : 0.0f;

    float best[RB];
    int index[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) best[b] = -INFINITY, index[b] = -1;
    const int4 zero = make_int4(0, 0, 0, 0);
    for (int chunk = c0; chunk < c1; ++chunk) {
        const int64_t base = static_cast<int64_t>(chunk) * kChunk;
        const uint32_t size = static_cast<uint32_t>(min(a.vocab - base, static_cast<int64_t>(kChunk)));
        const int valid = static_cast<int>(size) - mine;
        // (unsigned: tokens below the chunk, negative ones among them, lie past it)
        const auto place = [&](int token) { return static_cast<uint32_t>(token) - static_cast<uint32_t>(base); };
        *reinterpret_cast<int4*>(&seen_lds[mine]) = zero;
        *reinterpret_cast<int4*>(&entry_lds[mine]) = zero;
        if (paths) {
#pragma unroll
            for (int b = 0; b < RB; ++b) *reinterpret_cast<int4*>(&path_lds[b][mine]) = zero;
        }
        __syncthreads();
        for (int begin = 0; begin < history_n; begin += kVec * kChunk) {
            if (begin || (history_n > kVec * kChunk && chunk > c0)) {
                load_history(begin);
                cut_history(begin);
            }
#pragma unroll
            for (int u = 0; u < kVec; ++u) {
                if (begin + u * kChunk >= history_n) break;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t at = place(h[u][e]);
                    if (at < size) atomicAdd(&seen_lds[at], 1);
                }
            }
        }
        for (int i = tid; i < bias_n; i += kT) {
            const uint32_t at = place(i == tid ? first_bias : bias_tokens[i]);
            if (at < size) atomicMax(&entry_lds[at], i + 1);
        }
        int on_path = 0;
        for (int pair = tid; pair < pairs; pair += kT) {
            const uint32_t at = place(pair == tid ? first_path : path_token(pair));
            if (at < size) {
                atomicAdd(&path_lds[pair / nodes][at], 1);
                on_path = 1;
            }
        }
        on_path = __syncthreads_or(on_path);   // most chunks hold none of a path's tokens
        int seen[4];
        float bias[4];
        bool biased[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            seen[e] = seen_lds[mine + e];
            const int entry = entry_lds[mine + e];
            biased[e] = entry > 0;
            bias[e] = entry > 0 ? a.r.bias_values[seq * a.r.bias_stride + entry - 1] : 0.0f;
        }
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = x[b][e];
                const int n = seen[e] + (on_path ? path_lds[b][mine + e] : 0);
                if (n > 0) {
                    if (a.r.repetition) v = v > 0.0f ? v / rep : v * rep;
                    if (a.r.frequency) v = v - static_cast<float>(n) * freq;
                    if (a.r.presence) v = v - pres;
                }
                if (biased[e]) v = v + bias[e];
                if (!(allowed[b] >> e & 1)) v = -INFINITY;
                if (e < valid && v > best[b]) best[b] = v, index[b] = static_cast<int>(base) + mine + e;
                x[b][e] = v;
            }
        if (a.out && valid > 0) {
#pragma unroll
            for (int b = 0; b < RB; ++b)
                if (b < n_rows) store4(static_cast<T*>(a.out) + (row0 + b) * a.vocab + base + static_cast<int64_t>(mine), valid, x[b]);
        }
        if (chunk + 1 < c1) load_rows(chunk + 1);
    }
    if (!a.tokens) return;
    uint64_t key[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) key[b] = candidate(best[b], index[b]);
    wave_best(key);
    if ((tid & 63) == 0)
#pragma unroll
        for (int b = 0; b < RB; ++b) wave_key[b][tid >> 6] = key[b];
    __syncthreads();
    if (tid >= 64) return;
    // Lane r of the first wave finishes row r.
    bool last = false;
    if (tid < n_rows) {
        const int64_t row = row0 + tid;
        const uint64_t k = max(max(wave_key[tid][0], wave_key[tid][1]), max(wave_key[tid][2], wave_key[tid][3]));
        if (a.ranges == 1) {
            a.tokens[row] = candidate_token(k);
        } else {
            __hip_atomic_store(a.candidates + row * a.ranges + range, k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            publish_partials();
            last = ticket_take(a.tickets + row * kTicketStride, a.ranges) == static_cast<unsigned>(a.ranges - 1);
        }
    }
    // The wave together reduces the rows whose last range this was.
    for (uint64_t todo = __ballot(last); todo; todo &= todo - 1) {
        const int64_t row = row0 + __builtin_ctzll(todo);
        uint64_t k[1] = {0};
        for (int c = tid; c < a.ranges; c += 64) {
            uint64_t* from = a.candidates + row * a.ranges + c;
            k[0] = max(k[0], __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            // (zero again, as the workspace is between calls of any shapes)
            __hip_atomic_store(from, uint64_t(0), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        wave_best(k);
        if (tid == 0) {
            a.tokens[row] = candidate_token(k[0]);
            __hip_atomic_store(a.tickets + row * kTicketStride, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// Rows of a workgroup, and workgroups that share a row's vocabulary.
struct Plan {
    int row_batch, groups, chunks, ranges;
};

Plan plan(int64_t seqs, int64_t rows, int64_t vocab) {
    Plan p;
    p.row_batch = rows > 1 ? kRowBatch : 1;
    p.groups = static_cast<int>((rows + p.row_batch - 1) / p.row_batch);
    p.chunks = static_cast<int>((vocab + kChunk - 1) / kChunk);
    p.ranges = static_cast<int>(std::clamp<int64_t>(kTargetGroups / (seqs * p.groups), 1, p.chunks));
    return p;
}

int check_shape(int64_t seqs, int64_t rows, int64_t vocab) {
    if (seqs < 0 || rows < 0 || seqs > kMaxRows || rows > kMaxRows || seqs * rows > kMaxRows)
        return fail_inval("logits_rules: seqs * rows must be in [0, 65536]");
    if (vocab < 1 || vocab > 0x7fffffff) return fail_inval("logits_rules: vocab must be in [1, 2^31)");
    return 0;
}

template <typename T>
void launch(const Args& a, int row_batch, int64_t grid, hipStream_t stream) {
    if (row_batch == 1)
        hipLaunchKernelGGL((logits_rules_kernel<T, 1>), dim3(static_cast<unsigned>(grid)), dim3(kT), 0, stream, a);
    else
        hipLaunchKernelGGL((logits_rules_kernel<T, kRowBatch>), dim3(static_cast<unsigned>(grid)), dim3(kT), 0, stream, a);
}

}  // namespace
}  // namespace vmhip

using namespace vmhip;

extern "C" {

int64_t vm_hip_logits_rules_workspace_bytes(int64_t seqs, int64_t rows, int64_t vocab) {
    clear_error();
    VM_TRY(check_shape(seqs, rows, vocab));
    if (seqs * rows == 0) return 0;
    return seqs * rows * (kTicketStride * 4 + plan(seqs, rows, vocab).ranges * int64_t(8));
}

int vm_hip_logits_rules_apply(const vm_hip_logits_rules* rules, const void* logits, void* out, int dtype,
                              int32_t* tokens, int64_t seqs, int64_t rows, int64_t vocab, const int32_t* counts,
                              void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    VM_TRY(check_shape(seqs, rows, vocab));
    if (!rules) return fail_inval("logits_rules: null rules");
    if (dtype != VM_HIP_DTYPE_F32 && dtype != VM_HIP_DTYPE_F16 && dtype != VM_HIP_DTYPE_BF16)
        return fail_inval("logits_rules: dtype must be F32, F16 or BF16");
    if (rules->history && (!rules->history_lengths || rules->history_stride < 0 ||
                           rules->history_stride > kMaxList))
        return fail_inval("logits_rules: history needs its lengths and stride");
    if (rules->bias_tokens &&
        (!rules->bias_values || !rules->bias_lengths || rules->bias_stride < 0 || rules->bias_stride > kMaxList))
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
    const Plan p = plan(seqs, rows, vocab);
    a.tickets = static_cast<unsigned*>(workspace);
    a.candidates = tokens ? reinterpret_cast<uint64_t*>(a.tickets + seqs * rows * kTicketStride) : nullptr;
    a.vocab = vocab;
    a.rows = static_cast<int>(rows);
    a.words = static_cast<int>((rows + 63) / 64);
    a.mask_words = static_cast<int>((vocab + 31) / 32);
    a.chunks = p.chunks;
    a.groups = p.groups;
    a.ranges = p.ranges;
    const int64_t grid = seqs * p.groups * p.ranges;
    auto s = static_cast<hipStream_t>(stream);
    if (dtype == VM_HIP_DTYPE_F16)
        launch<F16>(a, p.row_batch, grid, s);
    else if (dtype == VM_HIP_DTYPE_BF16)
        launch<BF16>(a, p.row_batch, grid, s);
    else
        launch<float>(a, p.row_batch, grid, s);
    return check_launch("logits_rules", s);
}

}  // extern "C"
