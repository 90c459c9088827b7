// Causal attention of many requests in one call: over cache pages (decoded
// tokens and chunks of prompts) and of whole prompts that lie one behind the
// other.
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp(scale (q_r . k_j) - m_r),
//
// j over the tokens up to the row's own, m_r a reference that is at least the
// largest score less kHeadroom.  The query heads of a KV head read the same keys,
// so the (token, head) pairs of a request and KV head are its query rows, r =
// token G + head.  Both products are computed transposed, S^T = K Q^T and O^T =
// V^T P^T, so that a query row owns a column of both and its statistics stay in
// its lanes; keys are numbered inside a tile so that the scores a lane holds
// are the weights that the second product wants from it.
//
// Two kernels.  attention_few_kernel takes requests of at most 16 RT query
// rows (decoded tokens, where plan() does not leave them to the other): K and V straight from memory to operand registers, a
// wave its own blocks of keys, and the keys of all requests dealt out evenly
// over the workgroups.  attention_many_kernel takes the others: 32 RT rows a
// wave, key tiles in LDS for all four waves.  16-bit rows use the 16-bit matrix
// instructions (weights rounded to 16 bits: half a step of the rows' type for
// each, F16 as kLift says), fp32 rows the fp32 ones.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kv_paged.h"
#include "kv_q8.h"
#include "lds_load.h"
#include "vm_device.h"
#include "vm_internal.h"

namespace vmhip {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxBatch = VM_HIP_PAGED_MAX_BATCH;
constexpr int kMaxSplits = 64;        // workgroups that share a request's keys: few rows,
constexpr int kManySplits = 28;       // many rows
constexpr int kMaxShared = 1024;      // row tiles of a KV head that may share workgroups,
constexpr int kShareUnits = 2048;     // and of all
constexpr int kTargetGroups = 512;    // workgroups that fill 256 compute units twice
constexpr int kTicketStride = 16;     // a ticket has a 64-byte line of its own
constexpr int64_t kTicketBytes = kTargetGroups * kTicketStride * 4;
constexpr int kRound = 128;           // keys that the waves of attention_few_kernel take at once
// A weight may exceed 1 by this much (log2) before its row's reference moves:
// references then move in the first blocks and rarely later.
constexpr float kHeadroom = 7.0f;
// An exponent is one multiply-add, score times scale less the reference, whose
// rounding (2^-24 of the reference) all weights share.  Where a reference is 2^16
// or more, and it comes near a factor, the wave's scores lose theirs before they are
// scaled: such rows have the lowest limit, so that every block goes where references
// move.
constexpr float kFar = 65536.0f;
constexpr float kAlways = -3.402823466e38f;
// What a row's reference weighs (log2).  F16 weights below 2^-14 have an error of
// up to 2^-25 instead of half a step, below 2^-25 they are lost, and the sum of
// weights, in fp32, keeps them: behind a key that weighs 1, 100000 others of e^-17
// would count for half as much again.  The type goes to 65504, so its references
// weigh 2^8, weights with the headroom 2^15: errors are half a step down to 2^-22 of
// the reference and 2^-33 of it below.  All weights of a row are larger by the
// same, which its sum takes out again.
template <typename T>
constexpr float kLift = std::is_same<T, F16>::value ? 8.0f : 0.0f;

struct Args {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int32_t* row_start;
    const int32_t* lengths;   // with pages
    const int32_t* tables;
    unsigned* tickets;   // kTargetGroups
    char* parts;
    int64_t q_stride, k_stride, v_stride;   // elements
    int max_pages, pages;
    int batch, rows, max_rows, heads, kv_heads, shift;
    int few;       // query rows up to which a request is of few rows
    bool shared;   // whether a tile of many rows may have several workgroups
    int group;     // query heads of a KV head
    unsigned per_group;   // 2^32 / group, rounded up (group 1: not used)
    float c;   // scale / ln 2
};

// A request's rows and the tokens in front of them.
struct Request {
    int start, n, length, p0;   // first row, rows, tokens, tokens in front of the first row (negative: rows without)
    int todo;                   // rows that are computed
    bool falls;                 // the next offset is below this request's
};

// `falls`: some offset is below an earlier one, and the largest up to b counts
// (every row is one request's).  Offsets of a plan rise, and only the others pay
// for the walk.
template <bool kPaged>
__device__ __forceinline__ Request request(const Args& a, int b, bool falls) {
    Request r;
    int from = a.row_start[b];
    const int to = a.row_start[b + 1];
    r.falls = to < from;
    if (__builtin_expect(falls, false))
        for (int i = 0; i < b; ++i) from = max(from, a.row_start[i]);
    r.start = min(max(from, 0), a.rows);
    r.n = min(max(to, r.start), a.rows) - r.start;
    if (kPaged) {
        r.length = min(max(a.lengths[b], 0), a.max_pages << a.shift);
    } else {
        r.length = r.n;
    }
    r.p0 = r.length - r.n;
    r.todo = min(r.n, a.max_rows);
    return r;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Request uniform(const Request& r) {
    return {uniform(r.start), uniform(r.n), uniform(r.length), uniform(r.p0), uniform(r.todo), r.falls};
}

__device__ __forceinline__ float max_halves(float v) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    unsigned q[2];
    __builtin_memcpy(q, &h, sizeof q);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float sum_halves(float v) { return swap_halves_add(v, v); }
// Over the lanes lr + 16 g.
__device__ __forceinline__ float max_groups(float v) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    unsigned q[2];
    __builtin_memcpy(q, &p, sizeof q);
    return max_halves(fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1])));
}
__device__ __forceinline__ float sum_groups(float v) {
    v = swap_rows_add(v, v);
    return swap_halves_add(v, v);
}

// The rows' references, scaled; true: some row of the wave has a far one, and they
// are to be taken from the scores.
template <int RT>
__device__ __forceinline__ bool references(const float (&m)[RT], float c, float (&ref)[RT]) {
    bool far = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        ref[rt] = m[rt] * c;
        far |= !(fabsf(ref[rt]) < kFar);
    }
    if (__builtin_expect(__any(far) == 0, true)) return false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) ref[rt] = 0.0f;
    return true;
}

// Elements that are not finite: bits that odd_bits() leaves in kOddMask (adding
// one to an exponent of all ones carries into the sign's place), and a dword
// without them.
template <typename T>
constexpr uint32_t kExponent = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, F16>::value ? 0x7c007c00u : 0x7f807f80u;
template <typename T>
constexpr uint32_t kOddMask = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
template <typename T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t bits) {
    constexpr uint32_t kStep = kExponent<T> & ~(kExponent<T> << 1);   // the exponents' lowest bits
    return (bits & kExponent<T>) + kStep;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_elements(uint32_t bits) {
    const uint32_t odd = odd_bits<T>(bits) & kOddMask<T>;
    if constexpr (sizeof(T) == 4) return odd ? 0u : bits;
    if (odd & 0x8000u) bits &= 0xffff0000u;
    if (odd & 0x80000000u) bits &= 0x0000ffffu;
    return bits;
}

template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x4 x, u32x4 y, f32x4 z) {
    if constexpr (std::is_same<T, F16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), z, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, x), __builtin_bit_cast(bf8, y), z, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ f32x16 mfma32(u32x4 x, u32x4 y, f32x16 z) {
    if constexpr (std::is_same<T, F16>::value)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), z, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, x), __builtin_bit_cast(bf8, y), z, 0, 0, 0);
}

// Eight weights as an operand, rounded to nearest.
template <typename T>
__device__ __forceinline__ u32x4 pack8(const float* p) {
    if constexpr (std::is_same<T, F16>::value) {
        half8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = static_cast<_Float16>(p[e]);
        return __builtin_bit_cast(u32x4, h);
    } else {
        bf8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = static_cast<__bf16>(p[e]);
        return __builtin_bit_cast(u32x4, h);
    }
}

// The compiler moves vector and scalar arithmetic across this, nothing else.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0x406); }

__device__ __forceinline__ void store4(float* p, const float* y) { *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]); }
__device__ __forceinline__ void store4(F16* p, const float* y) {
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
    const half4 h{static_cast<_Float16>(y[0]), static_cast<_Float16>(y[1]), static_cast<_Float16>(y[2]), static_cast<_Float16>(y[3])};
    *reinterpret_cast<half4*>(p) = h;
}
__device__ __forceinline__ void store4(BF16* p, const float* y) {
    typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
    const bf4 h{static_cast<__bf16>(y[0]), static_cast<__bf16>(y[1]), static_cast<__bf16>(y[2]), static_cast<__bf16>(y[3])};
    *reinterpret_cast<bf4*>(p) = h;
}

// A query row's token and head of the group: rows are counted from the first
// of token t0, and are few (less than the group's size and 256).
struct Row {
    int t, head;
};
__device__ __forceinline__ Row row_of(const Args& a, int t0, int r) {
    // r / group as the upper half of r times 2^32 / group, rounded up
    const int t = static_cast<int>(__umulhi(static_cast<unsigned>(r), a.per_group)) + (a.group == 1 ? r : 0);
    return {t0 + t, r - t * a.group};
}

// One row's four dims: outputs over the sum of weights; a row that saw nothing: zeros.
template <typename T>
__device__ __forceinline__ void put(const Args& a, const Request& q, int kh, Row r, int dim, const float* y, float l, int d) {
    if (r.t >= q.todo) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float z[4] = {y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv};
    store4(static_cast<T*>(a.out) + (static_cast<int64_t>(q.start + r.t) * a.heads + kh * a.group + r.head) * d + dim, z);
}

struct RowDim {
    int row, dim;
};

// Parts of a tile's keys in the workspace: four outputs for each thread in turn
// (place(i): the row and first dim of the i-th), then references (log2) and sums
// of the rows; the workgroup that draws the last ticket joins them.  part(s):
// byte offset of workgroup s's; rows: how many the parts hold, mine: whether
// this wave's threads have any; factors: LDS for active x kRows floats, totals for
// kRows.
// kParts parts at a time and as many of a thread's items as make 16 loads in
// flight; the first are requested before the factors' inputs.
template <typename T, int D, int kRows, int kParts, typename Part, typename Place>
__device__ __forceinline__ void join_by(const Args& a, const Request& q, int kh, int t0, int r0, int active, int rows,
                                        bool mine, const char* parts, Part part, Place place, float* factors,
                                        float* totals) {
    constexpr int kItems = kRows * D / 4 / kThreads;
    constexpr int kTake = kItems < 16 / kParts ? kItems : 16 / kParts;
    static_assert(kItems % kTake == 0, "items are taken evenly");
    u32x4 x[kTake][kParts];
    const auto request_parts = [&](int i0, int s0) {
#pragma unroll
        for (int u = 0; u < kParts; ++u) {
            if (s0 + u >= active) break;
            const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(parts + part(s0 + u), kRows * D * 4);
#pragma unroll
            for (int i = 0; i < kTake; ++i) x[i][u] = coherent_load16(rs, ((i0 + i) * kThreads + threadIdx.x) * 16);
        }
    };
    if (mine) request_parts(0, 0);
    for (int row = threadIdx.x / 16; row < rows; row += kThreads / 16) {
        const int s0 = threadIdx.x % 16;
        float mv[kMaxSplits / 16], lv[kMaxSplits / 16], m = -INFINITY;
#pragma unroll
        for (int u = 0; u < kMaxSplits / 16; ++u) {
            const int s = s0 + 16 * u;
            const float* ml = reinterpret_cast<const float*>(parts + part(min(s, active - 1))) + kRows * D + row;
            mv[u] = s < active ? coherent_load(ml) : -INFINITY;
            lv[u] = s < active ? coherent_load(ml + kRows) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kMaxSplits / 16; ++u) m = fmaxf(m, mv[u]);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        const float m_ref = m == -INFINITY ? 0.0f : m;
        float l = 0.0f;
#pragma unroll
        for (int u = 0; u < kMaxSplits / 16; ++u) {
            const int s = s0 + 16 * u;
            const float f = __builtin_amdgcn_exp2f(mv[u] - m_ref);
            if (s < active) {
                l = fmaf(lv[u], f, l);
                factors[s * kRows + row] = f;
            }
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) l += __shfl_xor(l, o, 64);
        if (s0 == 0) totals[row] = l;
    }
    __syncthreads();
    if (!mine) return;
    for (int i0 = 0; i0 < kItems; i0 += kTake) {
        float y[kTake][4] = {};
        for (int s0 = 0; s0 < active; s0 += kParts) {
            if (i0 + s0 > 0) request_parts(i0, s0);
#pragma unroll
            for (int u = 0; u < kParts; ++u) {
                if (s0 + u >= active) break;
#pragma unroll
                for (int i = 0; i < kTake; ++i) {
                    const float f = factors[(s0 + u) * kRows + place(i0 + i).row];
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[i][e] = fmaf(__uint_as_float(x[i][u][e]), f, y[i][e]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kTake; ++i) {
            const RowDim at = place(i0 + i);
            put<T>(a, q, kh, row_of(a, t0, r0 + at.row), at.dim, y[i], totals[at.row], D);
        }
    }
}
template <typename T, int D, int kRows, typename Part, typename Place>
__device__ __forceinline__ void join_parts(const Args& a, const Request& q, int kh, int t0, int r0, int active, int rows,
                                           bool mine, const char* parts, Part part, Place place, float* factors,
                                           float* totals) {
    if (active <= 4 && kRows * D / 4 / kThreads > 8)
        join_by<T, D, kRows, 4>(a, q, kh, t0, r0, active, rows, mine, parts, part, place, factors, totals);
    else
        join_by<T, D, kRows, 8>(a, q, kh, t0, r0, active, rows, mine, parts, part, place, factors, totals);
}

constexpr int64_t part_bytes(int64_t rows, int64_t d) { return rows * (d + 2) * 4; }

// Clears the ticket and says whether this workgroup drew the last one.
__device__ __forceinline__ bool last_arrival(unsigned* counter, int active, unsigned* drawn) {
    publish_partials();
    __syncthreads();
    if (threadIdx.x == 0) *drawn = ticket_take(counter, active);
    __syncthreads();
    if (*drawn != static_cast<unsigned>(active - 1)) return false;
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

// Running sums, up to and with each of `count` things, of what size(i) says of
// them, by the whole workgroup; their total and the largest size.  Some size
// negative: the largest is kNoSums, and the sums are not valid.
constexpr int kNoSums = 0x7fffffff;
template <int kMost>
struct Sums {
    int upto[kMost];
    int waves[kWaves], most[kWaves];
    int falls;   // of requests: whether offsets do (here because scalar registers are short)
};
template <int kMost, typename Size>
__device__ __forceinline__ int sum_up(int count, Sums<kMost>& s, Size size, int* largest) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (count == 1) {   // (every thread writes the same)
        s.upto[0] = *largest = size(0);
        return *largest;
    }
    const int each = (count + kThreads - 1) / kThreads, i0 = threadIdx.x * each;
    int sum = 0, most = 0;
    for (int i = i0; i < min(i0 + each, count); ++i) {
        const int w = size(i);
        sum += w;
        most = w < 0 ? kNoSums : max(most, w);
        s.upto[i] = sum;
    }
    int run = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(run, o, 64);
        if (lane >= o) run += x;
        most = max(most, __shfl_xor(most, o, 64));
    }
    if (lane == 63) s.waves[wave] = run, s.most[wave] = most;
    __syncthreads();
    int before = run - sum, total = 0;
    most = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += s.waves[w];
        total += s.waves[w];
        most = max(most, s.most[w]);
    }
    *largest = most;
    for (int i = i0; i < min(i0 + each, count); ++i) s.upto[i] += before;
    __syncthreads();
    return total;
}
// The sums of size(request) over all requests, and whether offsets fall.
template <bool kPaged, typename Size>
__device__ __forceinline__ int sum_up_requests(const Args& a, Sums<kMaxBatch>& s, Size size, int* largest) {
    const int total = sum_up(a.batch, s, [&](int b) {
        const Request q = request<kPaged>(a, b, false);
        return a.batch > 1 && q.falls ? -1 : size(q);   // (one request's rows are nobody else's)
    }, largest);
    const bool falls = uniform(*largest) == kNoSums;
    s.falls = falls;   // (every thread writes the same)
    if (__builtin_expect(!falls, true)) return total;
    return sum_up(a.batch, s, [&](int b) { return size(request<kPaged>(a, b, true)); }, largest);
}
// The first whose running sum is above x.
template <int kMost>
__device__ __forceinline__ int first_above(const Sums<kMost>& s, int count, int x) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s.upto[mid] > x)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

// ---- Few rows: 16-wide tiles.  A[i][k] and B[k][j] of a 16x16x32 product
// sit in lane i (j) + 16 (k / 8), element k % 8; of a 16x16x4 fp32 product in lane
// i (j) + 16 k; D[i][j] in lane j + 16 (i / 4), element i % 4.
//   S^T  16 bits: tile bt (0, 1) of a 32-key block has key 8 (i / 4) + 4 bt + i %
//        4 in row i, so that lane group lg = lane / 16 holds keys 8 lg .. + 7;
//        fp32: one tile of 16 keys, in order, lane group lg holds keys 4 lg .. + 3
//   K    16 bytes a lane of its key's row, 64 adjacent bytes in four lanes
//   O^T  16 bits: row i of tile db is dim (D / 16) i + db: a lane reads D / 16
//        adjacent elements of each of its eight keys and transposes them with
//        byte permutes; fp32: tile 4 h + u has dim 64 h + 4 i + u: nothing moves
// K and V are read once and only used by one wave, so they skip LDS; a block's
// loads are requested a block ahead.
//
// MI355X, passes back to back: one token each of 32 requests over 1 to 8000
// tokens, 64 heads of 128 on 8, bf16: 151 us, 5.2 TB/s of K and V (a copy: 5.35),
// bound by HBM; 16 requests of 4 tokens over 6000: 69 us (of 2: 57); one request
// over 100000: 89 us, 4.6 TB/s, over 8000: 17 us.  One fp32 token of 32 heads of 64
// on 4 over 2000: 9.3 us: the launch and a chain of trips (lengths, table, keys,
// ticket, parts) of about a microsecond each.
template <int D, int RT>
struct FewShared {
    float merge_o[kWaves][16 * RT * D];
    float merge_m[kWaves][16 * RT], merge_l[kWaves][16 * RT];
    Sums<kMaxBatch> sums;   // rounds of a KV head
    unsigned ticket;
};

template <typename T, int D, int RT>
__device__ __forceinline__ void few_rows(const Args& a, int id, FewShared<D, RT>& sh) {
    constexpr bool kWide = sizeof(T) == 4;
    constexpr int KB = kWide ? 16 : 32;          // keys of a block
    constexpr int KPL = KB / 4;                  // of a lane
    constexpr int NT = KB / 16;                  // score tiles
    constexpr int KC = D * sizeof(T) / 64;       // 16-byte pieces of a key that a lane reads
    constexpr int ND = D / 16;                   // dim tiles
    constexpr int VW = ND * sizeof(T) / 4;       // dwords of a value's row that a lane reads
    constexpr int kRows = 16 * RT;
    auto& merge_o = sh.merge_o;
    auto& merge_m = sh.merge_m;
    auto& merge_l = sh.merge_l;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, lg = lane >> 4;
    const int g = a.group;
    const auto rounds_of = [&](const Request& q) {
        return q.todo > 0 && q.todo * g <= a.few ? max((q.length + kRound - 1) / kRound, 1) : 0;
    };

    // Rounds of all requests, summed up by every workgroup for itself.
    int longest;
    const int total = a.kv_heads * sum_up_requests<true>(a, sh.sums, rounds_of, &longest);
    // Shares: even, worth a workgroup (64 KB of keys and values or so; one fp32
    // token over 2000: 9.0 us with one round, 9.9 with two; one of 64 heads of 128
    // over 8000, bf16: 23 and 17, with four 18.7), and no more than kMaxSplits of a request's keys.
    const int per = max(max((total + kTargetGroups - 1) / kTargetGroups, kWide ? 1 : 2),
                        (longest + kMaxSplits - 2) / (kMaxSplits - 1));
    int pos = id * per;
    const int end = total - pos > per ? pos + per : total;   // (pos + per may pass 31 bits)

    while (pos < end) {
        // The request, KV head and rounds that this share goes on with.
        const int b = __builtin_amdgcn_readfirstlane(first_above(sh.sums, a.batch, pos / a.kv_heads));
        const Request q = uniform(request<true>(a, b, sh.sums.falls));
        const int rounds = rounds_of(q);
        const int request_start = (sh.sums.upto[b] - rounds) * a.kv_heads;
        const int kh = (pos - request_start) / rounds;
        const int unit_start = request_start + kh * rounds;
        const int first = pos - unit_start, last = min(rounds, end - unit_start);
        const int first_group = unit_start / per;
        const int active = (unit_start + rounds - 1) / per - first_group + 1;
        pos = unit_start + last;

        const int64_t row_bytes = D * sizeof(T);
        const char* kbase = static_cast<const char*>(a.k) + ((static_cast<int64_t>(kh) << a.shift) * row_bytes);
        const char* vbase = static_cast<const char*>(a.v) + ((static_cast<int64_t>(kh) << a.shift) * row_bytes);
        const int64_t page_bytes = (static_cast<int64_t>(a.kv_heads) << a.shift) * row_bytes;
        const int32_t* table = a.tables + static_cast<int64_t>(b) * a.max_pages;
        const int in_page = (1 << a.shift) - 1;
        const int last_page = max(q.length - 1, 0) >> a.shift;
        const int whole = min(q.p0 + 1, q.length);   // keys that every row sees

        // This wave's blocks: round r's keys are shared out in turn.
        constexpr int kStep = kRound / KB;   // blocks of a round
        const int block_end = min(last * kStep, (q.length + KB - 1) / KB);
        int block = first * kStep + wave;
        // (a block's keys have one page, or, of 16 tokens, two)
        const auto page_of = [&](int block, int octet) {
            return table[min((min(block, block_end - 1) * KB + octet) >> a.shift, last_page)];
        };
        const int k_at = kWide ? 0 : 8 * (lr / 4), v_at = KPL * lg;   // this lane's keys of a block
        const auto valid = [&](int id) { return id >= 0 && id < a.pages; };
        // Loads go on past the last block with that block again: without a
        // branch around them, waits need not be for all.
        u32x4 kreg[NT][KC];
        uint32_t vreg[KPL][VW];
        const auto load_keys = [&](int block, int id) {
            const int at = (min(block, block_end - 1) * KB + k_at) & in_page;
            const char* p = kbase + (valid(id) ? id : 0) * page_bytes + (at + (kWide ? lr : lr % 4)) * row_bytes + 16 * lg;
#pragma unroll
            for (int bt = 0; bt < NT; ++bt)
#pragma unroll
                for (int s = 0; s < KC; ++s) kreg[bt][s] = *reinterpret_cast<const u32x4*>(p + 4 * bt * row_bytes + 64 * s);
        };
        const auto load_values = [&](int block, int id) {
            const int at = (min(block, block_end - 1) * KB + v_at) & in_page;
            const char* p = vbase + (valid(id) ? id : 0) * page_bytes + at * row_bytes + (kWide ? 16 : 4 * VW) * lr;
#pragma unroll
            for (int j = 0; j < KPL; ++j) {
                if constexpr (VW == 2) {
                    const u32x2 x = *reinterpret_cast<const u32x2*>(p + j * row_bytes);
                    vreg[j][0] = x.x;
                    vreg[j][1] = x.y;
                } else {   // (fp32: rows of 64 dims apart, tiles 4 h + u)
#pragma unroll
                    for (int h = 0; h < VW / 4; ++h) {
                        const u32x4 x = *reinterpret_cast<const u32x4*>(p + j * row_bytes + 256 * h);
#pragma unroll
                        for (int e = 0; e < 4; ++e) vreg[j][4 * h + e] = x[e];
                    }
                }
            }
        };

        int id_k = 0, id_v = 0, next_k = 0, next_v = 0;
        if (block < block_end) {
            id_k = page_of(block, k_at);
            id_v = page_of(block, v_at);
            next_k = page_of(block + kWaves, k_at);
            next_v = page_of(block + kWaves, v_at);
            load_keys(block, id_k);
            load_values(block, id_v);
        }

        // Queries: in registers, or, where these do not do, in LDS (where the
        // outputs are merged later).
        constexpr bool kQueriesInLds = RT == 2 && D == 128;
        u32x4 qf[kQueriesInLds ? 1 : RT][kQueriesInLds ? 1 : KC];
        u32x4* q_lds = reinterpret_cast<u32x4*>(merge_o[0]) + lane;
        static_assert(RT * KC * 1024 <= static_cast<int>(sizeof merge_o), "queries fit");
        int limit_key[RT];   // the last key that the row sees
        if (kQueriesInLds) __syncthreads();   // (the last segment's merge has been read)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const Row r = row_of(a, 0, 16 * rt + lr);
            const bool row_ok = r.t < q.todo;
            limit_key[rt] = row_ok ? q.p0 + r.t : -1;
            const T* qp = static_cast<const T*>(a.q) + static_cast<int64_t>(q.start + (row_ok ? r.t : 0)) * a.q_stride +
                          (kh * g + r.head) * D;
#pragma unroll
            for (int s = 0; s < KC; ++s) {
                if (kQueriesInLds && s % kWaves != wave) continue;
                u32x4 x = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(qp) + 64 * s + 16 * lg);
                if (!row_ok) x = u32x4{0, 0, 0, 0};
                if constexpr (kQueriesInLds)
                    q_lds[(rt * KC + s) * 64] = x;
                else
                    qf[rt][s] = x;
            }
        }
        if (kQueriesInLds) __syncthreads();
        const auto query = [&](int rt, int s) {
            if constexpr (kQueriesInLds)
                return q_lds[(rt * KC + s) * 64];
            else
                return qf[rt][s];
        };
        f32x4 acc[RT][ND];
        float m_run[RT];   // the score that weighs 1
        float limit[RT];   // the score from which on it moves; -inf before the first key, or kAlways
        float l_run[RT];   // sum of this lane's keys' weights
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int db = 0; db < ND; ++db) acc[rt][db] = f32x4{0.f, 0.f, 0.f, 0.f};
            m_run[rt] = l_run[rt] = 0.0f;
            limit[rt] = -INFINITY;
        }

        for (; block < block_end; block += kWaves) {
            if (kQueriesInLds) asm volatile("" : : : "memory");   // (read again: not kept in registers)
            const bool there = valid(id_v);
            f32x4 st[RT][NT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int bt = 0; bt < NT; ++bt) st[rt][bt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KC; ++s)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const u32x4 x = query(rt, s);
#pragma unroll
                    for (int bt = 0; bt < NT; ++bt) {
                        if constexpr (kWide) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                st[rt][bt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kreg[bt][s][e]), __uint_as_float(x[e]),
                                                                                  st[rt][bt], 0, 0, 0);
                        } else {
                            st[rt][bt] = mfma16<T>(kreg[bt][s], x, st[rt][bt]);
                        }
                    }
                }
            load_keys(block + kWaves, next_k);
            const bool masked = (block + 1) * KB > whole || !__all(there);
            if (masked) {
                const int key0 = block * KB + v_at;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int j = 0; j < KPL; ++j)
                        if (!(there && key0 + j <= limit_key[rt])) st[rt][j / 4][j % 4] = -INFINITY;
            }
            float mt[RT];
            bool moves = false;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                mt[rt] = -INFINITY;
#pragma unroll
                for (int j = 0; j < KPL; ++j) mt[rt] = fmaxf(mt[rt], st[rt][j / 4][j % 4]);
                moves |= mt[rt] > limit[rt];
            }
            float ref[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) ref[rt] = m_run[rt] * a.c;
            if (__any(moves)) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const float most = max_groups(mt[rt]);
                    if (most > -INFINITY) {
                        const float m = limit[rt] == -INFINITY ? most : fmaxf(m_run[rt], most);
                        const float fall = __builtin_amdgcn_exp2f((m_run[rt] - m) * a.c);
                        if (limit[rt] > -INFINITY) {
                            l_run[rt] *= fall;
#pragma unroll
                            for (int db = 0; db < ND; ++db) acc[rt][db] *= fall;
                        }
                        m_run[rt] = m;
                        limit[rt] = fabsf(m * a.c) < kFar ? m + kHeadroom / a.c : kAlways;
                    }
                }
                if (references(m_run, a.c, ref)) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int bt = 0; bt < NT; ++bt) st[rt][bt] -= m_run[rt];
                }
            }
            float p[RT][KPL];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float base = ref[rt] - kLift<T>;
#pragma unroll
                for (int j = 0; j < KPL; ++j) {
                    p[rt][j] = __builtin_amdgcn_exp2f(fmaf(st[rt][j / 4][j % 4], a.c, -base));
                    l_run[rt] += p[rt][j];
                }
            }
            if (masked) {
                // Values that are not finite, where not every row sees them: to
                // the rows that do by hand, whatever their weight (0 times them
                // would not be 0).
                uint32_t odd = 0;
#pragma unroll
                for (int j = 0; j < KPL; ++j)
#pragma unroll
                    for (int u = 0; u < VW; ++u) odd |= odd_bits<T>(vreg[j][u]);
                if (__any((odd & kOddMask<T>) != 0)) {
#pragma unroll
                    for (int j = 0; j < KPL; ++j)
#pragma unroll
                        for (int u = 0; u < VW; ++u) vreg[j][u] = finite_elements<T>(vreg[j][u]);
                    for (int j = 0; j < KB; ++j) {
                        const int key = block * KB + j;
                        const int id = table[min(key >> a.shift, last_page)];
                        if (!valid(id)) continue;
                        const T* vp = reinterpret_cast<const T*>(vbase + id * page_bytes + (key & in_page) * row_bytes);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            if (key > limit_key[rt]) continue;
                            for (int e = 0; e < 4; ++e)
#pragma unroll
                                for (int db = 0; db < ND; ++db) {
                                    const float x = widen(vp[kWide ? 64 * (db / 4) + 16 * lg + 4 * e + db % 4 : ND * (4 * lg + e) + db]);
#pragma unroll
                                    for (int w = 0; w < 4; ++w)
                                        if (w == e && !(fabsf(x) < INFINITY)) acc[rt][db][w] += x;
                                }
                        }
                    }
                }
            }
            if constexpr (kWide) {
#pragma unroll
                for (int db = 0; db < ND; ++db)
#pragma unroll
                    for (int j = 0; j < KPL; ++j)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
                            acc[rt][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vreg[j][db]), p[rt][j], acc[rt][db], 0, 0, 0);
            } else {
                u32x4 pf[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) pf[rt] = pack8<T>(p[rt]);
#pragma unroll
                for (int db = 0; db < ND; ++db) {
                    u32x4 vf;
#pragma unroll
                    for (int jp = 0; jp < 4; ++jp)
                        vf[jp] = __builtin_amdgcn_perm(vreg[2 * jp + 1][db / 2], vreg[2 * jp][db / 2],
                                                       db % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) acc[rt][db] = mfma16<T>(vf, pf[rt], acc[rt][db]);
                }
            }
            load_values(block + kWaves, next_v);
            id_v = next_v;
            next_k = page_of(block + 2 * kWaves, k_at);
            next_v = page_of(block + 2 * kWaves, v_at);
        }

        // Every wave's (reference, sum, output) to LDS; then thread (row, four
        // dims) merges the four.
        __syncthreads();   // (the last segment's merge has been read)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float l = sum_groups(l_run[rt]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int u = 0; u < ND / 4; ++u) {
                    const int dim = kWide ? 64 * u + 16 * lg + 4 * e : ND * (4 * lg + e) + 4 * u;
                    const float y[4] = {acc[rt][4 * u][e], acc[rt][4 * u + 1][e], acc[rt][4 * u + 2][e], acc[rt][4 * u + 3][e]};
                    store4(merge_o[wave] + (16 * rt + lr) * D + dim, y);
                }
            if (lg == 0) {
                merge_m[wave][16 * rt + lr] = limit[rt] == -INFINITY ? -INFINITY : m_run[rt] * a.c - kLift<T>;
                merge_l[wave][16 * rt + lr] = l;
            }
        }
        __syncthreads();
        const auto part = [&](int s) {   // the first group's part is its second one
            return (static_cast<int64_t>(first_group + s) * 2 + (s == 0)) * part_bytes(kRows, D);
        };
        char* out_part = a.parts + (active > 1 ? part(id - first_group) : 0);
        const __amdgpu_buffer_rsrc_t prs = buffer_rsrc(out_part, part_bytes(kRows, D));
        for (int item = threadIdx.x; item < kRows * D / 4; item += kThreads) {
            const int row = item / (D / 4), d4 = item % (D / 4);
            float m = merge_m[0][row];
#pragma unroll
            for (int k = 1; k < kWaves; ++k) m = fmaxf(m, merge_m[k][row]);
            const float m_ref = m == -INFINITY ? 0.0f : m;
            float l = 0.0f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kWaves; ++k) {
                const float f = __builtin_amdgcn_exp2f(merge_m[k][row] - m_ref);
                l = fmaf(merge_l[k][row], f, l);
                const float4 o = *reinterpret_cast<const float4*>(&merge_o[k][row * D + 4 * d4]);
                y[0] = fmaf(o.x, f, y[0]);
                y[1] = fmaf(o.y, f, y[1]);
                y[2] = fmaf(o.z, f, y[2]);
                y[3] = fmaf(o.w, f, y[3]);
            }
            if (active == 1) {
                put<T>(a, q, kh, row_of(a, 0, row), 4 * d4, y, l, D);
                continue;
            }
            coherent_store16(prs, static_cast<uint32_t>(item) * 16,
                             u32x4{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])});
            if (d4 == 0) {
                float* ml = reinterpret_cast<float*>(out_part) + kRows * D;
                coherent_store(ml + row, m);
                coherent_store(ml + kRows + row, l);
            }
        }
        if (active > 1 && last_arrival(a.tickets + first_group * kTicketStride, active, &sh.ticket)) {
            static_assert(kMaxSplits * kRows <= kWaves * kRows * D, "factors fit");
            const auto place = [&](int i) {
                const int item = i * kThreads + static_cast<int>(threadIdx.x);
                return RowDim{item / (D / 4), 4 * (item % (D / 4))};
            };
            join_parts<T, D, kRows>(a, q, kh, 0, 0, active, kRows, true, a.parts, part, place, merge_o[0], merge_m[0]);
        }
    }
}

// ---- Many rows: 32-wide tiles, 32 RT query rows a wave, KT keys at a time in
// LDS for all four waves, the next tile's on their way into a second buffer.
// A[i][k] and B[k][j] of a 32x32x16 product sit in lane i (j) + 32 (k / 8), element k % 8; of
// a 32x32x2 fp32 product in lane i (j) + 32 k; D[i][j] in lane j + 32 (i / 4 %
// 2), element i % 4 + 4 (i / 8).  A lane of half lh = lane / 32 holds the
// scores of keys 8 a + 4 lh + b: as weights they are the second product's k
// positions if V^T's operand has the same keys there, which two transposing LDS
// reads of four keys give (16 bits), or plain reads (fp32).
//
// MI355X, passes back to back: 3 prompts, 12000 tokens in all, 64 heads of 128 on 8,
// bf16: 963 us, 948 TFLOP/s (a large product: 1150); one of 6500, 64 heads of 64
// on 8, f16: 380 us, 910 TFLOP/s; 500 tokens behind 30000, 32 heads of 128 on 8,
// f16: 297 us, 835 TFLOP/s, with 7 tokens of other requests over 22000 beside them
// 415 to 430; one fp32 prompt of 2000, 64 heads of 128: 536 us, 122 TFLOP/s (153).
// The matrix cores are busy 40 % of the cycles: what is left is softmax between
// the products of two waves a SIMD (without the loads 496 us where it takes 640,
// without barriers too 472, without exponentials 436).  Eight waves and 128 keys a
// tile: 743 us for 625; a tile's scores beside the weights of the one before:
// registers spill, 1310.  A single tile alone on its compute unit waits for its
// keys: about 1.4 us for 64 of 128 dims, twice what its products take.
template <typename T, int D>
struct Tile {
    static constexpr int KT = sizeof(T) == 4 ? 32 : 64;         // keys
    static constexpr int CH = D * sizeof(T) / 16;               // 16-byte pieces of a row
    static constexpr int PER = KT * CH / kThreads;              // pieces of a thread
    static constexpr int kBytes = KT * D * static_cast<int>(sizeof(T));
    // Which piece of a row lies where: pieces are exchanged so that the 16 rows
    // of keys, and the 4 (or, fp32, 2) rows of values, that are read at a time
    // lie in different banks (64 of 4 bytes).
    static __device__ __forceinline__ int swap_k(int row) { return CH == 8 ? row >> 1 & 7 : row & 15; }
    static __device__ __forceinline__ int swap_v(int row) {
        return sizeof(T) == 4 ? 8 * (row >> 2 & 1) : CH == 8 ? 4 * (row >> 1 & 1) : 4 * (row & 3);
    }
};

template <typename T, int D>
struct ManyShared {
    char tile[2][2][Tile<T, D>::kBytes];   // [buffer][keys, values]
    Sums<kMaxBatch> requests;              // tiles of a KV head
    Sums<kMaxShared> tiles;                // rounds of a KV head
    unsigned ticket;
};

template <typename T, int D, int RT, bool kPaged>
__device__ __forceinline__ void many_rows(const Args& a, int id, ManyShared<T, D>& sh) {
    constexpr bool kWide = sizeof(T) == 4;
    using L = Tile<T, D>;
    constexpr int KT = L::KT, CH = L::CH, PER = L::PER;
    constexpr int NK = KT / 32;             // score tiles
    constexpr int NQ = D * sizeof(T) / 32;  // 16-byte pieces of a query row that a lane holds
    constexpr int ND = D / 32;              // dim tiles
    constexpr int kRows = 32 * RT * kWaves;
    constexpr int kRowBytes = D * sizeof(T);
    constexpr int kLeastTiles = kWide ? 2 : 4;   // key tiles that are worth a workgroup
    constexpr int kAhead = 4;                    // LDS operands in front of their products
    constexpr int kJoin = kWide ? 6 : D == 64 ? 28 : 16;   // key tiles' time that all workgroups' parts take,
    constexpr int kJoinFew = kWide ? 6 : D == 64 ? 16 : 10;   // and those of fewer
    constexpr int kStart = kWide ? 1 : 2;        // key tiles' time that a row tile takes beside its keys

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lc = lane & 31, lh = lane >> 5;
    const int g = a.group;
    const auto tiles_of = [&](const Request& q) {
        const int r = q.todo * g;
        return r > a.few ? (r + kRows - 1) / kRows : 0;
    };
    constexpr int kLeast = kStart + kLeastTiles;

    int longest;
    const int tiles_all = sum_up_requests<kPaged>(a, sh.requests, tiles_of, &longest);
    if (tiles_all == 0) return;
    // A row tile's keys go to one workgroup, or all tiles' keys are dealt out
    // evenly (as attention_few_kernel's are), where the first would take longer
    // than dealing out and the storing and joining of the parts (512 workgroups'
    // 16-bit parts take 25 us: kJoin; less where the shares are the least that is
    // worth a workgroup and fewer take part: kJoinFew, 100 rows beside 7 tokens over
    // 2000, 32 heads of 64 on 8: 27.6 us, one workgroup a tile 38.9).  Times in key tiles of a compute unit:
    // up to 256 tiles have one each, up to 512 share one by twos (below), more
    // follow as others end (of tiles of equal length the last alone).  32 heads of 64
    // on 4, f16, 3000 rows: 55 us against 79 dealt out; 40 rows of 64 heads of 128 on
    // 8 behind 2000: 57 against 40, behind 1000: 36.5 against 39.5.
    const int units = tiles_all * a.kv_heads;
    bool shared = a.shared && tiles_all <= kMaxShared && units <= kShareUnits;
    int of_head = 0;
    if (shared) {
        of_head = sum_up(tiles_all, sh.tiles, [&](int i) {
            const int b = first_above(sh.requests, a.batch, i);
            const Request q = request<kPaged>(a, b, sh.requests.falls);
            const int r0 = (i - (sh.requests.upto[b] - tiles_of(q))) * kRows;
            const int seen = min(q.p0 + min((r0 + kRows - 1) / g, q.todo - 1) + 1, q.length);
            return kStart + max((seen + KT - 1) / KT, 1);
        }, &longest);
        const int each = of_head * a.kv_heads / kTargetGroups;
        const int alone = units <= kTargetGroups / 2 ? longest
                          : units <= kTargetGroups   ? max(longest, 2 * each)
                                                     : 2 * each + max(2 * (of_head / tiles_all) - longest, 0);
        shared = longest > kLeast && alone > 2 * max(each, kLeast) + (each >= kLeast ? kJoin : kJoinFew);
    }
    int pos = id, end = id + 1, share = 1;   // of the units (KV head, row tile), or of their key tiles
    if (shared) {
        const int total = of_head * a.kv_heads;
        share = max(max((total + kTargetGroups - 1) / kTargetGroups, kLeast), (longest + kManySplits - 2) / (kManySplits - 1));
        if (id >= kTargetGroups) return;
        // neighbours, which read the same keys, on one XCD
        id = id % 8 * (kTargetGroups / 8) + id / 8;
        pos = id * share;
        end = min(total, pos + share);
    } else {
        end = min(end, tiles_all * a.kv_heads);
    }

    // The tile with `rank` tiles in front of it that see more keys (of up to 64
    // requests, one a lane): tile t of a request sees about as many as tile t +
    // p0 group / kRows of a request without tokens in front.
    const auto by_length = [&](int rank) {
        const bool real = lane < a.batch;
        const Request q = request<kPaged>(a, real ? lane : 0, sh.requests.falls);
        const int mine = real ? tiles_of(q) : 0;
        const int ahead = static_cast<int>(static_cast<int64_t>(max(q.p0, 0)) * g / kRows);
        const int before = sh.requests.upto[real ? lane : 0] - mine;
        const auto from = [&](int level) {   // tiles of all requests from this level on
            int n = min(max(mine + ahead - level, 0), mine);
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o, 64);
            return uniform(n);
        };
        int lo = 0, hi = mine + ahead;       // from(lo) > rank >= from(hi)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) hi = max(hi, __shfl_xor(hi, o, 64));
        hi = uniform(hi);
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            if (from(mid) > rank)
                lo = mid;
            else
                hi = mid;
        }
        // the n-th of the requests that have a tile of this level
        uint64_t has = __ballot(lo >= ahead && lo < ahead + mine);
        for (int n = rank - from(lo + 1); n > 0; --n) has &= has - 1;
        const int b = has ? __builtin_ctzll(has) : 0;
        return __builtin_amdgcn_readlane(before + lo - ahead, b);
    };

    while (pos < end) {
        int kh, slot, first = 0, last = 0x7fffffff, active = 1, first_group = 0;
        if (shared) {
            kh = pos / of_head;
            slot = first_above(sh.tiles, tiles_all, pos - kh * of_head);
            const int before = slot ? sh.tiles.upto[slot - 1] : 0;
            const int size = sh.tiles.upto[slot] - before, start = kh * of_head + before;
            first = max(pos - start - kStart, 0);
            last = min(end - start, size) - kStart;
            first_group = (start + kStart) / share;
            active = (start + size - 1) / share - first_group + 1;
            pos = start + size;
            if (last <= first) continue;
        } else {
            // Workgroups go to the XCDs in turn, eight at a time: a KV head's tiles
            // stay on one where the count of those allows, those that see the most
            // keys first.  Of the 512 that start at once a compute unit has the n-th
            // and the 256 + n-th: the second half goes backwards.
            int at = pos / 8;
            const int half = kTargetGroups / 16, both = min(kTargetGroups, tiles_all * a.kv_heads) / 8;
            if (at >= half && at < both) at = half + both - 1 - at;
            if (a.kv_heads % 8 == 0) {
                slot = at % tiles_all;
                kh = at / tiles_all * 8 + pos % 8;
            } else {
                slot = (8 * at + pos % 8) / a.kv_heads;
                kh = (8 * at + pos % 8) % a.kv_heads;
            }
            // Of several requests, by length where that balances compute units (4 of
            // 4000 rows in all, 32 heads of 128 on 8, bf16: 64.6 us against 69.7);
            // of more tiles, a request's together for the caches' sake (3 of 12000
            // in all: 964 against 992).
            const bool sorted = a.batch > 1 && a.batch <= 64 && units > kTargetGroups / 2 && units <= 2 * kTargetGroups;
            slot = sorted ? by_length(uniform(slot)) : tiles_all - 1 - slot;
            pos = end;
        }
        kh = uniform(kh);
        first = uniform(first);
        last = uniform(last);
        active = uniform(active);
        first_group = uniform(first_group);
        const int b = uniform(first_above(sh.requests, a.batch, slot));
        const Request q = uniform(request<kPaged>(a, b, sh.requests.falls));
        const int r0 = uniform(slot - (sh.requests.upto[b] - tiles_of(q))) * kRows;
        const int t0 = r0 / g, rem0 = r0 - t0 * g;   // its token, and the rows of that in front
        const int t_last = min(uniform(row_of(a, t0, rem0 + kRows - 1).t), q.todo - 1);
        const int seen = min(max(q.p0 + t_last + 1, 0), q.length);      // keys that some row sees
        const int whole = min(max(q.p0 + t0 + 1, 0), q.length);         // that every row sees
        last = min(last, (seen + KT - 1) / KT);
        const int rows = min(q.todo * g - r0, kRows);
        const bool has_rows = 32 * RT * wave < rows;   // this wave

        // Where the tile's pieces lie: a wave's piece u is 1 KB, kWaveRows rows.
        constexpr int kWaveRows = 64 / CH, kStep = kWaves * kWaveRows;   // rows of a piece, of the waves' pieces u
        static_assert(kStep <= 32, "those rows lie in two 16-key groups at most");
        const int my_row = wave * kWaveRows + lane / CH;
        static_assert(kStep % 8 == 0, "pieces u and u + 2 of a lane are exchanged alike");
        const auto k_piece = [&](int u) { return 16 * ((lane % CH) ^ L::swap_k(my_row + u % 2 * kStep)); };
        const uint32_t v_piece = 16 * ((lane % CH) ^ L::swap_v(my_row));
        const int in_page = (1 << a.shift) - 1;
        const int last_page = max(q.length - 1, 0) >> a.shift;
        const int32_t* table = kPaged ? a.tables + static_cast<int64_t>(b) * a.max_pages : nullptr;
        const uint32_t page_bytes = kPaged ? static_cast<uint32_t>(a.kv_heads << a.shift) * kRowBytes : 0;
        const int k_row = kPaged ? kRowBytes : static_cast<int>(a.k_stride * sizeof(T));
        const int v_row = kPaged ? kRowBytes : static_cast<int>(a.v_stride * sizeof(T));
        const char* k_base = static_cast<const char*>(a.k) +
                             (kPaged ? static_cast<int64_t>(kh << a.shift) * kRowBytes
                                     : static_cast<int64_t>(q.start) * k_row + kh * kRowBytes);
        const char* v_base = static_cast<const char*>(a.v) +
                             (kPaged ? static_cast<int64_t>(kh << a.shift) * kRowBytes
                                     : static_cast<int64_t>(q.start) * v_row + kh * kRowBytes);
        // The pages of a tile's keys, one a lane for the 16 keys from 16 (lane % kGroups) on.
        constexpr int kGroups = KT / 16;
        constexpr unsigned kAll = (1u << kGroups) - 1;
        const auto lookup = [&](int t) {
            if constexpr (kPaged)
                return table[min((t * KT + 16 * (lane % kGroups)) >> a.shift, last_page)];
            else
                return 0;
        };
        const auto valid = [&](int id) { return !kPaged || static_cast<unsigned>(id) < static_cast<unsigned>(a.pages); };
        const uint32_t k_mine[2] = {static_cast<uint32_t>((kPaged ? my_row % 16 : my_row) * k_row + k_piece(0)),
                                    static_cast<uint32_t>((kPaged ? my_row % 16 : my_row) * k_row + k_piece(1))};
        const uint32_t v_mine = (kPaged ? my_row % 16 : my_row) * v_row + v_piece;
        const auto load = [&](int t, int ids) {
            char* kl = sh.tile[t & 1][0] + wave * 1024;
            char* vl = sh.tile[t & 1][1] + wave * 1024;
            if constexpr (kPaged) {
                const int pages = valid(ids) ? ids : 0;
#pragma unroll
                for (int u = 0; u < PER; ++u) {
                    const int group = u * kStep / 16 + (kStep > 16 ? wave / (kWaves / 2) : 0);
                    const uint32_t id = __builtin_amdgcn_readlane(pages, group);
                    const uint32_t at = ((t * KT + 16 * group) & in_page) + (kStep < 16 ? u * kStep % 16 : 0);
                    const uint64_t offset = static_cast<uint64_t>(id) * page_bytes + at * kRowBytes;
                    lds_load16(k_base + offset, k_mine[u % 2], kl + u * (kWaves * 1024));
                    lds_load16(v_base + offset, v_mine, vl + u * (kWaves * 1024));
                }
            } else {
                const char* kp = k_base + static_cast<int64_t>(t * KT) * k_row;
                const char* vp = v_base + static_cast<int64_t>(t * KT) * v_row;
                const int left = q.length - 1 - t * KT;   // the last row there is
                if (left >= KT - 1) {
#pragma unroll
                    for (int u = 0; u < PER; ++u) {
                        lds_load16(kp + u * kStep * k_row, k_mine[u % 2], kl + u * (kWaves * 1024));
                        lds_load16(vp + u * kStep * v_row, v_mine, vl + u * (kWaves * 1024));
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < PER; ++u) {
                        const int row = min(my_row + u * kStep, left);
                        lds_load16(kp, row * k_row + k_piece(u), kl + u * (kWaves * 1024));
                        lds_load16(vp, row * v_row + v_piece, vl + u * (kWaves * 1024));
                    }
                }
            }
        };
        // Waits for the wave's pieces of the tile and meets the other waves.  `ask`
        // (tiles that not every row sees whole): values that are not finite are
        // taken out; true: there were some.
        const auto arrive = [&](int t, bool ask) {
            wait_loads();
            if (ask) {
                uint32_t odd = 0;
#pragma unroll
                for (int u = 0; u < PER; ++u) {
                    u32x4* at = reinterpret_cast<u32x4*>(sh.tile[t & 1][1] + (u * kWaves + wave) * 1024 + lane * 16);
                    const u32x4 v = *at;
                    const uint32_t bits = (odd_bits<T>(v.x) | odd_bits<T>(v.y) | odd_bits<T>(v.z) | odd_bits<T>(v.w)) & kOddMask<T>;
                    if (bits)
                        *at = u32x4{finite_elements<T>(v.x), finite_elements<T>(v.y), finite_elements<T>(v.z), finite_elements<T>(v.w)};
                    odd |= bits;
                }
                return __syncthreads_or(odd != 0) != 0;
            }
            __syncthreads();
            return false;
        };

        int ids = lookup(first), next = lookup(first + 1);   // of the tile that is computed, and of the next one
        if (first < last) load(first, ids);

        u32x4 qf[RT][NQ];
        int limit_key[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const Row r = row_of(a, t0, rem0 + 32 * (RT * wave + rt) + lc);
            const bool row_ok = r.t < q.todo;
            limit_key[rt] = row_ok ? q.p0 + r.t : -1;
            const T* qp = static_cast<const T*>(a.q) + static_cast<int64_t>(q.start + (row_ok ? r.t : 0)) * a.q_stride +
                          (kh * g + r.head) * D;
#pragma unroll
            for (int s = 0; s < NQ; ++s) {
                qf[rt][s] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(qp) + 32 * s + 16 * lh);
                if (!row_ok) qf[rt][s] = u32x4{0, 0, 0, 0};
            }
        }
        // Keys below wave_whole are seen by every row of the wave, from wave_seen on by none.
        const int w0 = uniform(row_of(a, t0, rem0 + 32 * RT * wave).t), w1 = uniform(row_of(a, t0, rem0 + 32 * RT * (wave + 1) - 1).t);
        const int wave_whole = w0 < q.todo ? min(max(q.p0 + w0 + 1, 0), q.length) : 0;
        const int wave_seen = w0 < q.todo ? min(seen, max(q.p0 + min(w1, q.todo - 1) + 1, 0)) : 0;

        f32x16 acc[RT][ND];
        float m_run[RT], limit[RT], l_run[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int db = 0; db < ND; ++db)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[rt][db][e] = 0.0f;
            m_run[rt] = l_run[rt] = 0.0f;
            limit[rt] = -INFINITY;
        }

        const auto compute = [&](int t, bool masked, unsigned bits) {
            const char* kt = sh.tile[t & 1][0];
            const char* vt = sh.tile[t & 1][1];
            f32x16 st[RT][NK];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int n = 0; n < NK; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) st[rt][n][e] = 0.0f;
            // LDS reads run kAhead operands in front of their products: left to
            // itself, the compiler waits for each before the next.
            const auto key_piece = [&](int i) {   // of score tile i / NQ, 16-byte piece i % NQ
                const int row = 32 * (i / NQ) + lc;
                return *reinterpret_cast<const u32x4*>(kt + row * kRowBytes + 16 * ((2 * (i % NQ) + lh) ^ L::swap_k(row)));
            };
            u32x4 kf[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) kf[i] = key_piece(i);
            keep_order();
#pragma unroll
            for (int i = 0; i < NK * NQ; ++i) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if constexpr (kWide) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            st[rt][i / NQ] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                                __uint_as_float(kf[i % kAhead][e]), __uint_as_float(qf[rt][i % NQ][e]), st[rt][i / NQ], 0, 0, 0);
                    } else {
                        st[rt][i / NQ] = mfma32<T>(kf[i % kAhead], qf[rt][i % NQ], st[rt][i / NQ]);
                    }
                }
                if (i + kAhead < NK * NQ) kf[i % kAhead] = key_piece(i + kAhead);
                keep_order();
            }
            if (masked) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int n = 0; n < NK; ++n)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int key = t * KT + 32 * n + 8 * (e / 4) + 4 * lh + e % 4;
                            if (!(key <= limit_key[rt] && (bits >> (2 * n + e / 8) & 1))) st[rt][n][e] = -INFINITY;
                        }
            }
            float mt[RT];
            bool moves = false;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                mt[rt] = -INFINITY;
#pragma unroll
                for (int n = 0; n < NK; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) mt[rt] = fmaxf(mt[rt], st[rt][n][e]);
                moves |= mt[rt] > limit[rt];
            }
            float ref[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) ref[rt] = m_run[rt] * a.c;
            if (__any(moves)) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const float most = max_halves(mt[rt]);
                    if (most > -INFINITY) {
                        const float m = limit[rt] == -INFINITY ? most : fmaxf(m_run[rt], most);
                        const float fall = __builtin_amdgcn_exp2f((m_run[rt] - m) * a.c);
                        if (limit[rt] > -INFINITY) {
                            l_run[rt] *= fall;
#pragma unroll
                            for (int db = 0; db < ND; ++db)
#pragma unroll
                                for (int e = 0; e < 16; ++e) acc[rt][db][e] *= fall;
                        }
                        m_run[rt] = m;
                        limit[rt] = fabsf(m * a.c) < kFar ? m + kHeadroom / a.c : kAlways;
                    }
                }
                if (references(m_run, a.c, ref)) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int n = 0; n < NK; ++n) st[rt][n] -= m_run[rt];
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float base = ref[rt] - kLift<T>;
#pragma unroll
                for (int n = 0; n < NK; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(st[rt][n][e], a.c, -base));
                        st[rt][n][e] = p;
                        l_run[rt] += p;
                    }
            }
            if constexpr (kWide) {
                const auto value = [&](int i) {   // of score element i / ND, dim tile i % ND
                    const int e = i / ND;
                    const int row = 8 * (e / 4) + 4 * lh + e % 4;
                    const int c = 8 * (i % ND) + lc / 4;
                    return *reinterpret_cast<const float*>(vt + row * kRowBytes + 16 * (c ^ L::swap_v(row)) + 4 * (lc & 3));
                };
                float x[2 * kAhead];
#pragma unroll
                for (int i = 0; i < 2 * kAhead; ++i) x[i] = value(i);
                keep_order();
#pragma unroll
                for (int i = 0; i < 16 * NK * ND; ++i) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        acc[rt][i % ND] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i % (2 * kAhead)], st[rt][i / ND / 16][i / ND % 16],
                                                                               acc[rt][i % ND], 0, 0, 0);
                    if (i + 2 * kAhead < 16 * NK * ND) x[i % (2 * kAhead)] = value(i + 2 * kAhead);
                    if (i % 2) keep_order();
                }
            } else {
                const int l16 = lane & 15;
                const auto value_piece = [&](int i) {   // of 16 keys i / ND, dim tile i % ND
                    u32x4 x;
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        // lane 4 k + x of 16 reads dims 4 x .. + 3 of key k
                        const int row = 16 * (i / ND) + 8 * w + 4 * lh + l16 / 4;
                        const int c = 4 * (i % ND) + 2 * (lane >> 4 & 1) + (l16 % 4) / 2;
                        const char* at = vt + row * kRowBytes + 16 * (c ^ L::swap_v(row)) + 8 * (l16 & 1);
                        const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                                      (__attribute__((address_space(3))) s16x4*)(at)));
                        x[2 * w] = y.x;
                        x[2 * w + 1] = y.y;
                    }
                    return x;
                };
                u32x4 vf[kAhead], pf[RT];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) vf[i] = value_piece(i);
                keep_order();
#pragma unroll
                for (int i = 0; i < 2 * NK * ND; ++i) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        if (i % ND == 0) {
                            float p[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) p[e] = st[rt][i / ND / 2][i / ND % 2 * 8 + e];
                            pf[rt] = pack8<T>(p);
                        }
                        acc[rt][i % ND] = mfma32<T>(vf[i % kAhead], pf[rt], acc[rt][i % ND]);
                    }
                    if (i + kAhead < 2 * NK * ND) vf[i % kAhead] = value_piece(i + kAhead);
                    keep_order();
                }
            }
        };
        // The values of a tile that are not finite, to the rows that see them,
        // whatever their weight: 0 times them would not be 0.
        const auto add_odd = [&](int t, unsigned bits) {
            for (int j = 0; j < KT; ++j) {
                if (!(bits >> (j / 16) & 1)) continue;
                const int key = min(t * KT + j, q.length - 1);
                const char* row = v_base;
                if constexpr (kPaged)
                    row += static_cast<uint64_t>(static_cast<uint32_t>(table[key >> a.shift])) * page_bytes + (key & in_page) * kRowBytes;
                else
                    row += static_cast<int64_t>(key) * v_row;
                const T* vp = reinterpret_cast<const T*>(row) + 4 * lh;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (t * KT + j > limit_key[rt]) continue;
#pragma unroll
                    for (int db = 0; db < ND; ++db)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float x = widen(vp[32 * db + 8 * (e / 4) + e % 4]);
                            if (!(fabsf(x) < INFINITY)) acc[rt][db][e] += x;
                        }
                }
            }
        };

        for (int t = first; t < last; ++t) {
            const unsigned bits = __ballot(valid(ids)) & kAll;   // keys 16 u .. + 15 have a page
            const bool odd = arrive(t, (t + 1) * KT > whole || bits != kAll);
            // (the other buffer's tile is behind all waves)
            if (t + 1 < last) load(t + 1, next);
            ids = next;
            next = lookup(t + 2);
            if (t * KT >= wave_seen) continue;
            if (odd) add_odd(t, bits);
            compute(t, (t + 1) * KT > wave_whole || bits != kAll, bits);
        }

        const auto part = [&](int s) {   // the first group's part is its second one
            return (static_cast<int64_t>(first_group + s) * 2 + (s == 0)) * part_bytes(kRows, D);
        };
        const auto place = [&](int i) {   // i = 4 (ND rt + db) + u
            return RowDim{32 * (RT * wave + i / (4 * ND)) + lc, 8 * (i % (4 * ND)) + 4 * lh};
        };
        char* out_part = a.parts + (active > 1 ? part(id - first_group) : 0);
        const __amdgpu_buffer_rsrc_t prs = buffer_rsrc(out_part, part_bytes(kRows, D));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (!has_rows) break;
            const float l = sum_halves(l_run[rt]);
            const int row = 32 * (RT * wave + rt) + lc;
#pragma unroll
            for (int db = 0; db < ND; ++db)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float y[4] = {acc[rt][db][4 * u], acc[rt][db][4 * u + 1], acc[rt][db][4 * u + 2], acc[rt][db][4 * u + 3]};
                    const int i = 4 * (ND * rt + db) + u;
                    if (active == 1)
                        put<T>(a, q, kh, row_of(a, t0, rem0 + row), place(i).dim, y, l, D);
                    else
                        coherent_store16(prs, (i * kThreads + static_cast<int>(threadIdx.x)) * 16,
                                         u32x4{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])});
                }
            if (active > 1 && lh == 0) {
                float* ml = reinterpret_cast<float*>(out_part) + kRows * D;
                coherent_store(ml + row, limit[rt] == -INFINITY ? -INFINITY : m_run[rt] * a.c - kLift<T>);
                coherent_store(ml + kRows + row, l);
            }
        }
        __syncthreads();   // (LDS is free)
        if (active > 1 && last_arrival(a.tickets + first_group * kTicketStride, active, &sh.ticket)) {
            float* f = reinterpret_cast<float*>(sh.tile[0][0]);
            static_assert((kManySplits + 1) * kRows * 4 <= static_cast<int>(sizeof sh.tile), "factors fit");
            join_parts<T, D, kRows>(a, q, kh, t0, rem0, active, rows, has_rows, a.parts, part, place, f, f + kManySplits * kRows);
            __syncthreads();
        }
    }
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(kThreads, 2) void attention_few_kernel(const Args a) {
    __shared__ __align__(16) FewShared<D, RT> sh;
    few_rows<T, D, RT>(a, blockIdx.x, sh);
}
template <typename T, int D, int RT, bool kPaged>
__global__ __launch_bounds__(kThreads, 2) void attention_many_kernel(const Args a) {
    __shared__ __align__(16) ManyShared<T, D> sh;
    many_rows<T, D, RT, kPaged>(a, blockIdx.x, sh);
}

// ---- Host

struct Plan {
    bool few, many;
    int few_tiles;        // RT of attention_few_kernel
    int few_rows;         // query rows up to which a request is its
    int many_tiles;       // RT of attention_many_kernel
    bool shared;          // whether a request's keys may go to several workgroups
    int64_t many_groups;
    int64_t bytes;        // of the parts; the kernels run one after the other
};

// The bytes grow with rows and max_rows: a workspace serves smaller calls too.
Plan plan(int64_t batch, int64_t rows, int64_t max_rows, int64_t heads, int64_t kv_heads, int64_t d,
          int64_t max_tokens, bool wide, bool paged) {
    Plan p{};
    const int64_t g = heads / kv_heads;
    const int64_t most = std::min(rows, max_rows > 0 ? max_rows : rows) * g;   // query rows of a request
    // (requests between 17 and 32 rows are the other kernel's where that runs anyway)
    p.few_tiles = most <= 16 || (most > 32 && g <= 16) ? 1 : 2;
    p.few_rows = 16 * p.few_tiles;
    // Where some request is known to have more rows than that, 16-bit calls are the
    // other kernel's altogether: tokens then run beside the chunk instead of before
    // it (16 bits, 32 heads of 128 on 8: a chunk of 500 behind 30000 beside 7 tokens
    // 430 us against 456, of 11 behind 769 beside 4 27.6 against 41.4).  fp32 tokens
    // would take the matrix cores from it (100 rows beside 31 tokens over 2000, 32
    // heads of 64 on 4: 91 us against 71).  Rows not known: most calls hold tokens
    // alone, which are this kernel's (32 over 8000, 64 heads of 128 on 8: 151 us
    // against 157, one over 2000, 32 of 64: 7.6 against 34.5).
    p.few = paged && g <= p.few_rows && (most <= p.few_rows || (batch > 1 && (wide || max_rows == 0)));
    if (!p.few) p.few_rows = 0;
    p.many = most > p.few_rows;
    p.shared = max_tokens > kRound;
    if (p.few && p.shared) p.bytes = 2 * kTargetGroups * part_bytes(32, d);
    if (p.many) {
        // Two row tiles a wave read a key tile's operands once for both, where
        // registers allow, enough tiles are left for the workgroups and the tile's
        // tokens are few (f16, 64 heads of 64 on 8, 6500 rows: 380 us against 414; 32
        // on 4, 3000 rows: 75 against 55; 32 on 32, 6000 rows: 227 against 195).
        p.many_tiles = d == 64 && !wide && g >= 4 && rows * g / 256 * kv_heads >= kTargetGroups ? 2 : 1;
        const int64_t tile = 32 * p.many_tiles * kWaves;
        const int64_t units = (rows * g / tile + batch) * kv_heads;   // at most
        p.many_groups = p.shared ? std::max<int64_t>(units, kTargetGroups) : units;
        if (p.shared) p.bytes = 2 * kTargetGroups * part_bytes(d == 64 ? 256 : 128, d);
    }
    return p;
}

int check_call(const char* who, int64_t batch, int64_t rows, int64_t max_rows, int64_t heads, int64_t kv_heads,
               int64_t d) {
    const std::string w(who);
    if (d != 64 && d != 128) return fail_inval(w + ": head_dim must be 64 or 128");
    if (batch < 0 || batch > kMaxBatch || rows < 0 || rows > VM_HIP_PAGED_MAX_ROWS || max_rows < 0)
        return fail_inval(w + ": batch or rows out of range");
    if (kv_heads < 1 || kv_heads > 4096 || heads < 1 || heads > 65536 || heads % kv_heads || heads / kv_heads > 4096)
        return fail_inval(w + ": bad heads");
    if (rows * heads >= (int64_t{1} << 30)) return fail_inval(w + ": too many rows for one call");
    return 0;
}

int64_t workspace_bytes_of(int64_t batch, int64_t rows, int64_t max_rows, int64_t heads, int64_t kv_heads, int64_t d,
                           int64_t max_tokens, bool paged) {
    if (batch == 0 || rows == 0) return 0;
    const Plan p = plan(batch, rows, max_rows, heads, kv_heads, d, max_tokens, false, paged);
    return kTicketBytes + p.bytes;   // (the same for every type)
}

template <typename T, int D, bool kPaged>
void launch_type(const Args& a, const Plan& p, hipStream_t s) {
    const dim3 block(kThreads), few(kTargetGroups), many(static_cast<unsigned>(p.many_groups));
    if constexpr (kPaged) {
        if (p.few && p.few_tiles == 1)
            hipLaunchKernelGGL((attention_few_kernel<T, D, 1>), few, block, 0, s, a);
        else if (p.few)
            hipLaunchKernelGGL((attention_few_kernel<T, D, 2>), few, block, 0, s, a);
    }
    if (!p.many) return;
    if constexpr (D == 64 && sizeof(T) == 2) {
        if (p.many_tiles == 2) {
            hipLaunchKernelGGL((attention_many_kernel<T, D, 2, kPaged>), many, block, 0, s, a);
            return;
        }
    }
    hipLaunchKernelGGL((attention_many_kernel<T, D, 1, kPaged>), many, block, 0, s, a);
}

template <bool kPaged>
int run(const char* who, Args a, const Plan& p, int dtype, int64_t d, void* workspace, void* stream) {
    a.few = p.few_rows;
    a.group = a.heads / a.kv_heads;
    a.per_group = static_cast<unsigned>(((uint64_t{1} << 32) + a.group - 1) / a.group);
    a.shared = p.shared;
    a.tickets = static_cast<unsigned*>(workspace);
    a.parts = static_cast<char*>(workspace) + kTicketBytes;
    auto s = static_cast<hipStream_t>(stream);
    if (d == 64) {
        if (dtype == VM_HIP_DTYPE_F32)
            launch_type<float, 64, kPaged>(a, p, s);
        else if (dtype == VM_HIP_DTYPE_F16)
            launch_type<F16, 64, kPaged>(a, p, s);
        else
            launch_type<BF16, 64, kPaged>(a, p, s);
    } else {
        if (dtype == VM_HIP_DTYPE_F32)
            launch_type<float, 128, kPaged>(a, p, s);
        else if (dtype == VM_HIP_DTYPE_F16)
            launch_type<F16, 128, kPaged>(a, p, s);
        else
            launch_type<BF16, 128, kPaged>(a, p, s);
    }
    return check_launch(who, s);
}

float scale_of(float scale, int64_t d) {
    return (scale > 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(d))) * 1.44269504f;
}

// The factor that the kernels multiply scores by (scale / ln 2) has to be finite as well.
int check_scale(const char* who, float scale, int64_t d) {
    if (!(scale < INFINITY) || !(scale_of(scale, d) < INFINITY))
        return fail_inval(std::string(who) + ": scale must be finite, also divided by ln 2");
    return 0;
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
bool off4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) != 0; }

}  // namespace
}  // namespace vmhip

using namespace vmhip;

extern "C" {

int64_t vm_hip_attention_packed_workspace_bytes(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                                int64_t head_dim) {
    clear_error();
    VM_TRY(check_call("attention_packed", batch, rows, 0, heads, kv_heads, head_dim));
    return workspace_bytes_of(batch, rows, 0, heads, kv_heads, head_dim, rows, false);
}

int vm_hip_attention_packed(const void* q, const void* k, const void* v, void* out, int dtype, int64_t q_stride,
                            int64_t k_stride, int64_t v_stride, int64_t batch, int64_t rows, int64_t heads,
                            int64_t kv_heads, int64_t head_dim, const int32_t* row_start, float scale, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    clear_error();
    if (dtype != VM_HIP_DTYPE_F32 && dtype != VM_HIP_DTYPE_F16 && dtype != VM_HIP_DTYPE_BF16)
        return fail_inval("attention_packed: dtype must be F32, F16 or BF16");
    VM_TRY(check_call("attention_packed", batch, rows, 0, heads, kv_heads, head_dim));
    const int64_t unit = dtype == VM_HIP_DTYPE_F32 ? 4 : 8;   // elements of 16 bytes
    for (int64_t s : {q_stride, k_stride, v_stride})
        if (s % unit || s > (1 << 22))
            return fail_inval("attention_packed: strides must be multiples of 16 bytes, at most 2^22 elements");
    if (q_stride < heads * head_dim || k_stride < kv_heads * head_dim || v_stride < kv_heads * head_dim)
        return fail_inval("attention_packed: strides must hold a row's heads");
    VM_TRY(check_scale("attention_packed", scale, head_dim));
    if (rows == 0 || batch == 0) return 0;
    if (!q || !k || !v || !out || !row_start) return fail_inval("attention_packed: null pointer");
    if (off16(q) || off16(k) || off16(v) || off16(out))
        return fail_inval("attention_packed: q, k, v and out must be 16-byte aligned");
    if (off4(row_start)) return fail_inval("attention_packed: row_start must be 4-byte aligned");
    const int64_t need = vm_hip_attention_packed_workspace_bytes(batch, rows, heads, kv_heads, head_dim);
    if (need > 0 && (!workspace || workspace_bytes < need || off16(workspace)))
        return fail_inval("attention_packed: workspace smaller than vm_hip_attention_packed_workspace_bytes or unaligned");
    const Plan p = plan(batch, rows, 0, heads, kv_heads, head_dim, rows, dtype == VM_HIP_DTYPE_F32, false);
    if (p.many_groups >= (1 << 24)) return fail_inval("attention_packed: too many rows for one call");
    Args a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.row_start = row_start;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.batch = static_cast<int>(batch);
    a.rows = a.max_rows = static_cast<int>(rows);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.c = scale_of(scale, head_dim);
    return run<false>("attention_packed", a, p, dtype, head_dim, workspace, stream);
}

int64_t vm_hip_attention_paged_workspace_bytes(int64_t batch, int64_t rows, int64_t max_rows, int64_t heads,
                                               int64_t kv_heads, int64_t head_dim, int64_t max_tokens) {
    clear_error();
    VM_TRY(check_call("attention_paged", batch, rows, max_rows, heads, kv_heads, head_dim));
    if (max_tokens < 1 || max_tokens > (1 << 24)) return fail_inval("attention_paged: max_tokens out of range");
    return workspace_bytes_of(batch, rows, max_rows, heads, kv_heads, head_dim, max_tokens, true);
}

int vm_hip_attention_paged(const vm_hip_kv_paged* cache, const int32_t* tables, int64_t max_pages, const void* q,
                           void* out, int64_t batch, int64_t rows, int64_t max_rows, int64_t heads,
                           const int32_t* row_start, const int32_t* lengths, float scale, void* workspace,
                           int64_t workspace_bytes, void* stream) {
    clear_error();
    VM_TRY(check_kv_paged(cache, "attention_paged"));
    const int64_t d = cache->head_dim, hk = cache->kv_heads;
    VM_TRY(check_call("attention_paged", batch, rows, max_rows, heads, hk, d));
    if (max_pages < 1 || max_pages > (1 << 24) / cache->page_size)
        return fail_inval("attention_paged: max_pages * page_size must be at most 2^24");
    // (attention_few_kernel rounds the requests' rounds up to workgroups in 32 bits)
    if (batch * hk * ((max_pages * cache->page_size + kRound - 1) / kRound) > 0x7fffffff - (kTargetGroups - 1))
        return fail_inval("attention_paged: batch * kv_heads * max_pages * page_size must be at most 2^38 - 2^16");
    VM_TRY(check_scale("attention_paged", scale, d));
    if (rows == 0 || batch == 0) return 0;
    if (!tables || !q || !out || !row_start || !lengths) return fail_inval("attention_paged: null pointer");
    if (off16(q) || off16(out)) return fail_inval("attention_paged: q and out must be 16-byte aligned");
    if (off4(tables) || off4(row_start) || off4(lengths))
        return fail_inval("attention_paged: tables, row_start and lengths must be 4-byte aligned");
    const int64_t tokens = max_pages * cache->page_size;
    const int64_t need = vm_hip_attention_paged_workspace_bytes(batch, rows, max_rows, heads, hk, d, tokens);
    if (need > 0 && (!workspace || workspace_bytes < need || off16(workspace)))
        return fail_inval("attention_paged: workspace smaller than vm_hip_attention_paged_workspace_bytes or unaligned");
    const Plan p = plan(batch, rows, max_rows, heads, hk, d, tokens, cache->dtype == VM_HIP_DTYPE_F32, true);
    if (p.many_groups >= (1 << 24)) return fail_inval("attention_paged: too many rows for one call");
    Args a{};
    a.q = q;
    a.k = cache->k;
    a.v = cache->v;
    a.out = out;
    a.row_start = row_start;
    a.lengths = lengths;
    a.tables = tables;
    a.q_stride = heads * d;
    a.max_pages = static_cast<int>(max_pages);
    a.pages = static_cast<int>(cache->pages);
    a.batch = static_cast<int>(batch);
    a.rows = static_cast<int>(rows);
    a.max_rows = static_cast<int>(max_rows > 0 ? std::min(max_rows, rows) : rows);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(hk);
    a.shift = log2_of(cache->page_size);
    a.c = scale_of(scale, d);
    return run<true>("attention_paged", a, p, cache->dtype, d, workspace, stream);
}

}  // extern "C"
