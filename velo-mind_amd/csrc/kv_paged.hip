// A step over requests that share a pool of cache pages, without the
// attention (attention_paged.hip): the step's plan, pages given back, tables
// of the rotation, and the projection's rows on their way into the cache.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kv_paged.h"
#include "kv_q8.h"
#include "vm_device.h"
#include "vm_internal.h"

namespace vmhip {

int check_page_size(int64_t page_size, const char* who) {
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
        return fail_inval(std::string(who) + ": page_size must be 16, 32, 64, 128 or 256");
    return 0;
}

int check_kv_paged(const vm_hip_kv_paged* c, const char* who) {
    const std::string w(who);
    if (!c) return fail_inval(w + ": null cache");
    if (c->dtype != VM_HIP_DTYPE_F32 && c->dtype != VM_HIP_DTYPE_F16 && c->dtype != VM_HIP_DTYPE_BF16)
        return fail_inval(w + ": dtype must be F32, F16 or BF16");
    if (c->head_dim != 64 && c->head_dim != 128) return fail_inval(w + ": head_dim must be 64 or 128");
    VM_TRY(check_page_size(c->page_size, who));
    if (c->kv_heads < 1 || c->kv_heads > 4096 || c->pages < 1 || c->pages > 0x7fffffff / c->page_size)
        return fail_inval(w + ": pages or kv_heads out of range");
    if (!c->k || !c->v) return fail_inval(w + ": null cache pointer");
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
        return fail_inval(w + ": cache must be 16-byte aligned");
    return 0;
}

namespace {

constexpr int kT = 256;
constexpr int kMaxBatch = VM_HIP_PAGED_MAX_BATCH;

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
bool off4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) != 0; }
bool known_dtype(int d) { return d == VM_HIP_DTYPE_F32 || d == VM_HIP_DTYPE_F16 || d == VM_HIP_DTYPE_BF16; }

// Sums of non-negative numbers that stop at `cap` (half of what N holds at most):
// the order of the additions does not matter, and nothing leaves N.
template <typename N>
__device__ __forceinline__ N add_capped(N a, N b, N cap) { return min(a + b, cap); }

// The capped sum of the values of the threads in front of this one, and of all.
template <typename N>
__device__ __forceinline__ N sum_before(N v, N cap, N* waves, N* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const N o = __shfl_up(v, s, 64);
        if (lane >= s) v = add_capped(v, o, cap);
    }
    __syncthreads();   // (the sums of an earlier call have been read)
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    const N left = __shfl_up(v, 1, 64);
    N before = lane ? left : 0, total = 0;
#pragma unroll
    for (int w = 0; w < kT / 64; ++w) {
        if (w < wave) before = add_capped(before, waves[w], cap);
        total = add_capped(total, waves[w], cap);
    }
    *all = total;
    return before;
}

// The last index of start[0 .. n - 1] (non-decreasing, start[0] <= x) whose
// value is at most x.
template <typename N>
__device__ __forceinline__ int last_at_most(const N* start, int n, N x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// ---- The plan.  Every workgroup sums all requests up for itself (E
// consecutive ones a thread; 2048 requests are 16 KB, read from L2) and then
// places a row a thread: a search in LDS, one page id, two stores.  One launch
// and no second pass, because a page that is handed out starts with a row of
// this step: the row at its first position writes the table's entry.  The
// pool's count and the lengths may be updated in place: then the workgroup that
// draws the last ticket, when all have read them, writes both.  Bound by the
// launch and three round trips (requests, page ids, stores): 32 rows of 32
// requests 3.8 us, 128000 of 256 6.7 (four rows a thread: 9.3).
struct PlanArgs {
    vm_hip_page_plan p;
    int shift;          // log2 of the page size
    unsigned* ticket;   // with more than one workgroup and results in place
};

template <int E>
__global__ __launch_bounds__(kT) void kv_paged_plan_kernel(const PlanArgs a) {
    __shared__ int row_start[kMaxBatch + 1];   // rows in front of a request's
    __shared__ int page_start[kMaxBatch];      // pages handed out in front of a request's
    __shared__ int lengths[kMaxBatch];
    __shared__ int waves[kT / 64];
    __shared__ int handed_out;
    __shared__ unsigned drawn;
    const vm_hip_page_plan& p = a.p;
    const int batch = static_cast<int>(p.batch), rows = static_cast<int>(p.rows);
    const int page = 1 << a.shift;
    const int64_t longest = p.max_pages << a.shift;
    const int free_pages = min(max(*p.free_count, 0), static_cast<int>(p.pages));
    const int b0 = threadIdx.x * E;

    int length[E], count[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        length[e] = b0 + e < batch ? p.lengths[b0 + e] : 0;
        count[e] = b0 + e < batch ? p.counts[b0 + e] : 0;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        // A request that is too long for its table (or not valid) waits.
        if (length[e] < 0 || count[e] < 0 || static_cast<int64_t>(length[e]) + count[e] > longest) count[e] = 0;
        sum = add_capped(sum, min(count[e], rows + 1), rows + 1);
    }
    // Requests wait from the first whose rows do not fit.
    int all;
    int run = sum_before(sum, rows + 1, waves, &all);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        run = add_capped(run, min(count[e], rows + 1), rows + 1);
        if (run > rows) count[e] = 0;
    }
    // Pages: a request that wants more than are left waits, and so does every
    // later one that wants any.
    int want[E], wanted = 0;
    const int cap = free_pages + 1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int held = (max(length[e], 0) + page - 1) >> a.shift;
        want[e] = count[e] > 0 ? static_cast<int>((static_cast<int64_t>(length[e]) + count[e] + page - 1) >> a.shift) - held : 0;
        want[e] = min(want[e], cap);
        wanted = add_capped(wanted, want[e], cap);
    }
    int taken = 0, mine = 0;
    run = sum_before(wanted, cap, waves, &all);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int after = add_capped(run, want[e], cap);
        if (want[e] > 0 && after > free_pages) count[e] = want[e] = 0;
        if (b0 + e < batch) page_start[b0 + e] = run;
        if (want[e] > 0) taken = after;
        mine += count[e];
        run = after;
    }
    int total;
    run = sum_before(mine, 0x3fffffff, waves, &total);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (b0 + e < batch) row_start[b0 + e] = run, lengths[b0 + e] = length[e];
        run += count[e];
    }
    if (threadIdx.x == 0) row_start[batch] = total, handed_out = 0;
    __syncthreads();
    if (taken > 0) atomicMax(&handed_out, taken);
    __syncthreads();

    const int r = static_cast<int>(blockIdx.x) * kT + threadIdx.x;
    if (r < total) {
        const int b = last_at_most(row_start, batch, r);
        const int n = lengths[b];
        const int position = n + r - row_start[b];
        const int held = (n + page - 1) >> a.shift, at = position >> a.shift;
        int32_t* entry = p.tables + static_cast<int64_t>(b) * p.max_pages + at;
        const int id = at < held ? *entry : p.free_pages[free_pages - 1 - (page_start[b] + at - held)];
        if (at >= held && (position & (page - 1)) == 0) *entry = id;
        p.positions[r] = position;
        p.slots[r] = id >= 0 && id < p.pages ? (id << a.shift) + (position & (page - 1)) : -1;
    } else if (r < rows) {
        p.positions[r] = p.slots[r] = -1;
    }
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= batch; b += kT) p.row_start[b] = row_start[b];
    if (!a.ticket) {
        if (blockIdx.x != 0) return;
    } else if (gridDim.x > 1) {
        __syncthreads();   // this workgroup has read the lengths and the count
        if (threadIdx.x == 0) drawn = ticket_take(a.ticket, gridDim.x);
        __syncthreads();
        if (drawn != gridDim.x - 1) return;
        if (threadIdx.x == 0) __hip_atomic_store(a.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (b0 + e < batch) p.lengths_out[b0 + e] = length[e] + count[e];
    if (threadIdx.x == 0) *p.free_count_out = free_pages - handed_out;
}

// ---- Pages given back: one workgroup, E requests a thread summed up, then kRun
// adjacent entries a thread and step.  Entries that are no page are cleared but not
// given back (a plan would hand them out), so a step counts the others before it
// stores them; a pool that is full takes no more.  Sums are 64 bits: requests whose
// lengths are not valid hold whole tables.  A launch and four round trips for up to
// 2048 pages (5 of 256 requests, 2500 pages: 3.3 us), three more for each further
// 2048 (all 128000 pages of those: 213 us).
template <int E>
__global__ __launch_bounds__(kT) void kv_paged_release_kernel(int batch, int64_t max_pages, int64_t pages, int shift,
                                                              const int32_t* __restrict__ finished, int32_t* lengths,
                                                              int32_t* tables, int32_t* free_pages,
                                                              int32_t* free_count) {
    constexpr int kRun = 8;
    __shared__ int64_t start[kMaxBatch + 1];   // entries in front of a request's
    __shared__ int64_t waves[kT / 64];
    __shared__ int valid_waves[kT / 64];
    int64_t left = min(max(*free_count, 0), static_cast<int>(pages));
    const int b0 = threadIdx.x * E;
    int64_t n[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        n[e] = 0;
        if (b0 + e < batch && finished[b0 + e]) {
            const int64_t held = (static_cast<int64_t>(max(lengths[b0 + e], 0)) + (1 << shift) - 1) >> shift;
            n[e] = min(held, max_pages);
            lengths[b0 + e] = 0;
        }
        sum += n[e];
    }
    int64_t all;
    int64_t at = sum_before<int64_t>(sum, INT64_MAX / 2, waves, &all);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (b0 + e < batch) start[b0 + e] = at;
        at += n[e];
    }
    if (threadIdx.x == 0) start[batch] = all;
    __syncthreads();
    for (int64_t i0 = 0; i0 < all; i0 += kT * kRun) {
        const int64_t i = i0 + threadIdx.x * kRun;
        int id[kRun], valid = 0;
        int32_t* entry[kRun];
        int b = i < all ? last_at_most(start, batch, i) : 0;
#pragma unroll
        for (int u = 0; u < kRun; ++u) {
            id[u] = -1;
            if (i + u >= all) continue;
            while (start[b + 1] <= i + u) ++b;   // (start[batch] is above)
            entry[u] = tables + b * max_pages + (i + u - start[b]);
            id[u] = *entry[u];
        }
#pragma unroll
        for (int u = 0; u < kRun; ++u) valid += id[u] >= 0 && id[u] < pages;
        int given;
        int64_t to = left + sum_before<int>(valid, kT * kRun, valid_waves, &given);
#pragma unroll
        for (int u = 0; u < kRun; ++u) {
            if (i + u >= all) continue;
            *entry[u] = -1;
            if (id[u] < 0 || id[u] >= pages) continue;
            if (to < pages) free_pages[to] = id[u];
            ++to;
        }
        left = min(left + given, pages);
    }
    if (threadIdx.x == 0) *free_count = static_cast<int>(left);
}

// ---- Tables of the rotation.  Angles of far positions need 64 bits (131071
// radians leave 2^-7 of a turn in fp32): the first of a thread's R rows takes
// a sine and cosine in fp64, of its part of a turn, the others turn it on by the
// frequency's own, four products a row (each adds 2^-52 or so).  Pairs are
// adjacent lanes.  Bound by the stores (131072 rows of 64 pairs: 12.2 us, 5.5
// TB/s); small tables by the launch and one sine (2000 of 32: 4.5).
constexpr int kMaxPairs = 64;

struct RopeArgs {
    double turns[kMaxPairs], c[kMaxPairs], s[kMaxPairs];   // of a position: turns, cosine and sine
    double factor;
    float* cos_t;
    float* sin_t;
    int64_t first, rows;
    int pairs;
};

template <int R>
__global__ __launch_bounds__(kT) void rope_tables_kernel(const RopeArgs a) {
    const int64_t u = static_cast<int64_t>(blockIdx.x) * kT + threadIdx.x;
    const int64_t r0 = u / a.pairs * R;
    const int i = static_cast<int>(u % a.pairs);
    if (r0 >= a.rows) return;
    double s, c;
    const double t = static_cast<double>(a.first + r0) * a.turns[i];
    sincospi(2.0 * (t - rint(t)), &s, &c);
    c *= a.factor;
    s *= a.factor;
    const double tc = a.c[i], ts = a.s[i];
#pragma unroll
    for (int k = 0; k < R; ++k) {
        if (r0 + k >= a.rows) return;
        a.cos_t[(r0 + k) * a.pairs + i] = static_cast<float>(c);
        a.sin_t[(r0 + k) * a.pairs + i] = static_cast<float>(s);
        const double n = c * tc - s * ts;
        s = s * tc + c * ts;
        c = n;
    }
}

// ---- Norm, rotation and append.  Sixteen lanes own one head row of one
// token, V = D / 16 adjacent elements each: the sum of squares is four DPP
// steps away, pairs of the interleaved layout are a lane's own, and those of
// halves are exchanged through LDS (any even number of rotated elements does).
// A group takes the heads h0, h0 + step, ... of its token, with the table's
// row and the norms' weights in registers and the next head's row on its way.
// Bound: one read of qkv, one write of q, keys and values (4000 rows of 80 heads
// of 128, bf16, normed, half of each rotated in pairs: 36 us, 4.6 TB/s, a large
// copy 4.9 to 5.3; one row of 40 heads of 64: 3.7).
template <typename T, int N>
struct alignas(sizeof(T) * N >= 16 ? 16 : sizeof(T) * N) Vec {
    T e[N];
};

// Stores past the L2 cache: whatever reads them next runs on other XCDs as well,
// and the rows that are still read keep their place (4000 rows of 80 heads of
// 128, inputs not in a cache: 36 us against 39).
template <typename V>
__device__ __forceinline__ void store_past(V* p, const V& x) {
    typedef uint32_t Word __attribute__((ext_vector_type(sizeof(V) >= 16 ? 4 : sizeof(V) / 4)));
    constexpr int kWords = sizeof(V) / sizeof(Word);
    Word w[kWords];
    __builtin_memcpy(w, &x, sizeof(V));
#pragma unroll
    for (int i = 0; i < kWords; ++i) __builtin_nontemporal_store(w[i], reinterpret_cast<Word*>(p) + i);
}

struct AppendArgs {
    const void* qkv;
    void* q_out;
    void* k_out;      // rows, or pages
    void* v_out;      // pages; NULL: rows, values stay where they are
    const float* q_norm;
    const float* k_norm;
    const float* cos_t;
    const float* sin_t;
    const int32_t* positions;
    const int32_t* slots;
    int64_t rows, table_rows, slot_count;
    float eps;
    int heads, kv_heads, rotary, shift, step;
};

__device__ __forceinline__ float sum16(float v) {
    const auto ror = [](float x, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    v += ror(v, std::integral_constant<int, 0x121>{});
    v += ror(v, std::integral_constant<int, 0x122>{});
    v += ror(v, std::integral_constant<int, 0x124>{});
    v += ror(v, std::integral_constant<int, 0x128>{});
    return v;
}

template <typename T, int D, bool kPairs, bool kNorm>
__global__ __launch_bounds__(kT) void kv_paged_append_kernel(const AppendArgs a) {
    constexpr int N = D / 16;
    __shared__ float swap[kPairs ? 1 : kT / 16][kPairs ? 1 : D];
    const int group = threadIdx.x / 16, i = threadIdx.x & 15;
    const int64_t u = static_cast<int64_t>(blockIdx.x) * (kT / 16) + group;
    const int64_t token = u / a.step;
    if (token >= a.rows) return;   // whole groups leave
    const int position = a.positions[token];
    const int slot = a.slots ? a.slots[token] : 0;
    if (position < 0 || slot < 0 || slot >= a.slot_count) return;
    const int all = a.heads + (a.v_out ? 2 : 1) * a.kv_heads;
    const int width = a.heads + 2 * a.kv_heads;
    const int half = a.rotary / 2;
    const int64_t turn = min(static_cast<int64_t>(position), a.table_rows - 1) * half;

    float c[N], s[N];   // of the element's pair; 1, 0 past the rotated ones
    int partner[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int at = i * N + e;
        const int pair = kPairs ? at / 2 : at < half ? at : at - half;
        const bool turned = at < a.rotary;
        c[e] = turned ? a.cos_t[turn + pair] : 1.0f;
        s[e] = turned ? a.sin_t[turn + pair] : 0.0f;
        const bool upper = kPairs ? at & 1 : at >= half;
        if (!upper) s[e] = -s[e];
        partner[e] = !turned ? at : upper ? at - half : at + half;
    }
    float qw[N], kw[N];
    if (kNorm) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            qw[e] = a.q_norm[i * N + e];
            kw[e] = a.k_norm[i * N + e];
        }
    }
    const T* src = static_cast<const T*>(a.qkv) + token * width * D + i * N;
    const int h0 = static_cast<int>(u % a.step);
    Vec<T, N> next = *reinterpret_cast<const Vec<T, N>*>(src + static_cast<int64_t>(h0) * D);
    for (int h = h0; h < all; h += a.step) {
        Vec<T, N> x = next;
        next = *reinterpret_cast<const Vec<T, N>*>(src + static_cast<int64_t>(min(h + a.step, all - 1)) * D);
        T* dst;
        if (h < a.heads) {
            dst = static_cast<T*>(a.q_out) + (token * a.heads + h) * D;
        } else {
            const bool value = h >= a.heads + a.kv_heads;
            const int kh = h - a.heads - (value ? a.kv_heads : 0);
            T* base = static_cast<T*>(value ? a.v_out : a.k_out);
            if (a.slots)
                base += ((((static_cast<int64_t>(slot) >> a.shift) * a.kv_heads + kh) << a.shift) +
                         (slot & ((1 << a.shift) - 1))) * D;
            else
                base += (token * a.kv_heads + kh) * D;
            dst = base;
        }
        if (h < a.heads + a.kv_heads) {
            float y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = widen(x.e[e]);
            if (kNorm) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < N; ++e) sum = fmaf(y[e], y[e], sum);
                const float r = 1.0f / sqrtf(sum16(sum) * (1.0f / D) + a.eps);
#pragma unroll
                for (int e = 0; e < N; ++e) y[e] = y[e] * r * (h < a.heads ? qw[e] : kw[e]);
            }
            float other[N];
            if (kPairs) {
#pragma unroll
                for (int e = 0; e < N; ++e) other[e] = y[e ^ 1];
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) swap[group][i * N + e] = y[e];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int e = 0; e < N; ++e) other[e] = swap[group][partner[e]];
                __builtin_amdgcn_wave_barrier();
            }
            // (elements that are not rotated have no partner to take an infinity from)
#pragma unroll
            for (int e = 0; e < N; ++e)
                x.e[e] = narrow<T>(i * N + e < a.rotary ? fmaf(y[e], c[e], other[e] * s[e]) : y[e]);
        }
        store_past(reinterpret_cast<Vec<T, N>*>(dst + i * N), x);
    }
}

template <typename T, int D>
void launch_append(const AppendArgs& a, bool pairs, hipStream_t stream) {
    const int64_t groups = a.rows * a.step;
    const dim3 grid(static_cast<unsigned>((groups + kT / 16 - 1) / (kT / 16))), block(kT);
    if (a.q_norm) {
        if (pairs)
            hipLaunchKernelGGL((kv_paged_append_kernel<T, D, true, true>), grid, block, 0, stream, a);
        else
            hipLaunchKernelGGL((kv_paged_append_kernel<T, D, false, true>), grid, block, 0, stream, a);
    } else if (pairs) {
        hipLaunchKernelGGL((kv_paged_append_kernel<T, D, true, false>), grid, block, 0, stream, a);
    } else {
        hipLaunchKernelGGL((kv_paged_append_kernel<T, D, false, false>), grid, block, 0, stream, a);
    }
}

int append(const char* who, AppendArgs a, int dtype, int64_t heads, int64_t kv_heads, int64_t head_dim,
           const vm_hip_qk_norm* norm, const vm_hip_rope* rope, void* stream) {
    const std::string w(who);
    if (a.rows < 0 || a.rows > VM_HIP_PAGED_MAX_ROWS || heads < 1 || heads > 65536 || heads % kv_heads)
        return fail_inval(w + ": bad rows or heads");
    if (a.rows == 0) return 0;
    if (!a.qkv || !a.q_out || !a.k_out || !a.positions) return fail_inval(w + ": null pointer");
    if (off16(a.qkv) || off16(a.q_out) || off16(a.k_out))
        return fail_inval(w + ": qkv and the outputs must be 16-byte aligned");
    if (off4(a.positions) || off4(a.slots)) return fail_inval(w + ": positions and slots must be 4-byte aligned");
    if (norm) {
        if (!norm->q_weight || !norm->k_weight || off4(norm->q_weight) || off4(norm->k_weight))
            return fail_inval(w + ": null or unaligned norm weights");
        if (!(norm->eps >= 0.0f) || !std::isfinite(norm->eps)) return fail_inval(w + ": bad eps");
        a.q_norm = norm->q_weight;
        a.k_norm = norm->k_weight;
        a.eps = norm->eps;
    }
    bool pairs = false;
    if (rope) {
        if (rope->dim < 0 || rope->dim > head_dim || rope->dim % 2)
            return fail_inval(w + ": rotated elements must be even and at most head_dim");
        if (rope->layout != VM_HIP_ROPE_HALVES && rope->layout != VM_HIP_ROPE_PAIRS)
            return fail_inval(w + ": unknown rotation layout");
        if (rope->dim > 0) {
            if (rope->rows < 1 || !rope->cos_table || !rope->sin_table || off4(rope->cos_table) || off4(rope->sin_table))
                return fail_inval(w + ": rotation tables of no rows, null or unaligned");
            a.cos_t = rope->cos_table;
            a.sin_t = rope->sin_table;
            a.table_rows = rope->rows;
            a.rotary = static_cast<int>(rope->dim);
            pairs = rope->layout == VM_HIP_ROPE_PAIRS;
        }
    }
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    // Groups of a token: one a head while they do not fill the GPU, so that no
    // head waits for another (65536 of them instead of 16384: 2000 fp32 rows of 40
    // heads of 64 11.8 us, 8.4).
    const int all = a.heads + 2 * a.kv_heads;
    a.step = static_cast<int>(std::min<int64_t>(all, std::max<int64_t>(1, 16384 / a.rows)));
    auto s = static_cast<hipStream_t>(stream);
    if (head_dim == 64) {
        if (dtype == VM_HIP_DTYPE_F32)
            launch_append<float, 64>(a, pairs, s);
        else if (dtype == VM_HIP_DTYPE_F16)
            launch_append<F16, 64>(a, pairs, s);
        else
            launch_append<BF16, 64>(a, pairs, s);
    } else {
        if (dtype == VM_HIP_DTYPE_F32)
            launch_append<float, 128>(a, pairs, s);
        else if (dtype == VM_HIP_DTYPE_F16)
            launch_append<F16, 128>(a, pairs, s);
        else
            launch_append<BF16, 128>(a, pairs, s);
    }
    return check_launch(who, s);
}

}  // namespace
}  // namespace vmhip

using namespace vmhip;

extern "C" {

int64_t vm_hip_kv_paged_plan_workspace_bytes(int64_t batch, int64_t rows) {
    clear_error();
    if (batch < 0 || batch > kMaxBatch || rows < 0 || rows > VM_HIP_PAGED_MAX_ROWS)
        return fail_inval("kv_paged_plan: batch or rows out of range");
    return 64;
}

int vm_hip_kv_paged_plan(const vm_hip_page_plan* plan, void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    if (!plan) return fail_inval("kv_paged_plan: null plan");
    const vm_hip_page_plan& p = *plan;
    VM_TRY(check_page_size(p.page_size, "kv_paged_plan"));
    const int64_t need = vm_hip_kv_paged_plan_workspace_bytes(p.batch, p.rows);
    if (need < 0) return static_cast<int>(need);
    if (p.max_pages < 1 || p.max_pages > 0x7fffffff / p.page_size || p.pages < 1 || p.pages > 0x7fffffff / p.page_size)
        return fail_inval("kv_paged_plan: pages or max_pages out of range");
    if (p.batch == 0) return 0;
    const void* all[] = {p.lengths, p.counts, p.free_pages, p.free_count, p.tables, p.row_start, p.lengths_out,
                         p.free_count_out};
    for (const void* x : all)
        if (!x || off4(x)) return fail_inval("kv_paged_plan: null or unaligned pointer");
    if (p.rows > 0 && (!p.positions || !p.slots || off4(p.positions) || off4(p.slots)))
        return fail_inval("kv_paged_plan: null or unaligned pointer");
    if (!workspace || workspace_bytes < need || off16(workspace))
        return fail_inval("kv_paged_plan: workspace smaller than vm_hip_kv_paged_plan_workspace_bytes or unaligned");
    const bool in_place = p.lengths_out == p.lengths || p.free_count_out == p.free_count;
    PlanArgs a{p, log2_of(p.page_size), in_place ? static_cast<unsigned*>(workspace) : nullptr};
    const dim3 grid(static_cast<unsigned>(std::max<int64_t>(1, (p.rows + kT - 1) / kT))), block(kT);
    auto s = static_cast<hipStream_t>(stream);
    if (p.batch <= kT)
        hipLaunchKernelGGL(kv_paged_plan_kernel<1>, grid, block, 0, s, a);
    else if (p.batch <= 4 * kT)
        hipLaunchKernelGGL(kv_paged_plan_kernel<4>, grid, block, 0, s, a);
    else
        hipLaunchKernelGGL(kv_paged_plan_kernel<kMaxBatch / kT>, grid, block, 0, s, a);
    return check_launch("kv_paged_plan", s);
}

int vm_hip_kv_paged_release(int64_t batch, int64_t max_pages, int64_t pages, int64_t page_size, const int32_t* finished,
                            int32_t* lengths, int32_t* tables, int32_t* free_pages, int32_t* free_count, void* stream) {
    clear_error();
    VM_TRY(check_page_size(page_size, "kv_paged_release"));
    if (batch < 0 || batch > kMaxBatch || max_pages < 1 || max_pages > 0x7fffffff / page_size || pages < 1 ||
        pages > 0x7fffffff / page_size)
        return fail_inval("kv_paged_release: batch, pages or max_pages out of range");
    if (batch == 0) return 0;
    const void* all[] = {finished, lengths, tables, free_pages, free_count};
    for (const void* x : all)
        if (!x || off4(x)) return fail_inval("kv_paged_release: null or unaligned pointer");
    auto s = static_cast<hipStream_t>(stream);
    const int shift = log2_of(page_size), b = static_cast<int>(batch);
    if (batch <= kT)
        hipLaunchKernelGGL(kv_paged_release_kernel<1>, dim3(1), dim3(kT), 0, s, b, max_pages, pages, shift, finished,
                           lengths, tables, free_pages, free_count);
    else
        hipLaunchKernelGGL(kv_paged_release_kernel<kMaxBatch / kT>, dim3(1), dim3(kT), 0, s, b, max_pages, pages, shift, finished,
                           lengths, tables, free_pages, free_count);
    return check_launch("kv_paged_release", s);
}

int vm_hip_rope_tables(float* cos_table, float* sin_table, int64_t first, int64_t rows, int64_t dim, double theta,
                       const vm_hip_rope_scaling* scaling, void* stream) {
    clear_error();
    if (dim < 2 || dim > 2 * kMaxPairs || dim % 2) return fail_inval("rope_tables: dim must be even, 2 to 128");
    if (first < 0 || rows < 0 || first > (int64_t{1} << 31) || rows > (int64_t{1} << 31) - first)
        return fail_inval("rope_tables: positions must be below 2^31");
    if (!(theta > 1.0) || !std::isfinite(theta)) return fail_inval("rope_tables: theta must be above 1 and finite");
    RopeArgs a;
    a.factor = 1.0;
    const int kind = scaling ? scaling->kind : VM_HIP_ROPE_PLAIN;
    if (kind < VM_HIP_ROPE_PLAIN || kind > VM_HIP_ROPE_RAMP) return fail_inval("rope_tables: unknown scaling");
    if (scaling) {
        if (!(scaling->attention > 0.0) || !std::isfinite(scaling->attention))
            return fail_inval("rope_tables: attention factor must be positive and finite");
        a.factor = scaling->attention;
    }
    if (kind != VM_HIP_ROPE_PLAIN && (!(scaling->factor > 0.0) || !std::isfinite(scaling->factor)))
        return fail_inval("rope_tables: factor must be positive and finite");
    if (kind >= VM_HIP_ROPE_BANDS) {
        if (!(scaling->low > 0.0) || !(scaling->high > scaling->low) || !std::isfinite(scaling->high) ||
            !(scaling->original > 0.0) || !std::isfinite(scaling->original))
            return fail_inval("rope_tables: 0 < low < high and original > 0 are needed");
    }
    if (rows == 0) return 0;
    if (!cos_table || !sin_table || off4(cos_table) || off4(sin_table))
        return fail_inval("rope_tables: null or unaligned pointer");
    const double two_pi = 6.283185307179586476925286766559;
    double low = 0.0, high = 0.0;
    if (kind == VM_HIP_ROPE_RAMP) {
        // the pair that turns `turns` times in the trained length
        const auto pair_of = [&](double turns) {
            return dim * std::log(scaling->original / (turns * two_pi)) / (2.0 * std::log(theta));
        };
        low = std::max(std::floor(pair_of(scaling->high)), 0.0);
        high = std::min(std::ceil(pair_of(scaling->low)), static_cast<double>(dim - 1));
    }
    a.pairs = static_cast<int>(dim / 2);
    for (int i = 0; i < a.pairs; ++i) {
        double f = std::pow(theta, -2.0 * i / static_cast<double>(dim));
        if (kind == VM_HIP_ROPE_LINEAR) {
            f /= scaling->factor;
        } else if (kind == VM_HIP_ROPE_BANDS) {
            const double turns = scaling->original * f / two_pi;
            const double keep = std::min(1.0, std::max(0.0, (turns - scaling->low) / (scaling->high - scaling->low)));
            f = f * keep + f / scaling->factor * (1.0 - keep);
        } else if (kind == VM_HIP_ROPE_RAMP) {
            const double r = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
            f = f / scaling->factor * r + f * (1.0 - r);
        }
        a.turns[i] = f / two_pi;
        a.c[i] = std::cos(f);
        a.s[i] = std::sin(f);
    }
    a.cos_t = cos_table;
    a.sin_t = sin_table;
    a.first = first;
    a.rows = rows;
    auto s = static_cast<hipStream_t>(stream);
    // Four rows a thread while sixteen would leave the GPU idle.
    const int64_t r = rows * a.pairs >= (1 << 21) ? 16 : 4;
    const int64_t threads = (rows + r - 1) / r * a.pairs;
    const dim3 grid(static_cast<unsigned>((threads + kT - 1) / kT)), block(kT);
    if (r == 16)
        hipLaunchKernelGGL(rope_tables_kernel<16>, grid, block, 0, s, a);
    else
        hipLaunchKernelGGL(rope_tables_kernel<4>, grid, block, 0, s, a);
    return check_launch("rope_tables", s);
}

int vm_hip_kv_paged_append(const vm_hip_kv_paged* cache, const void* qkv, int64_t rows, int64_t heads,
                           const vm_hip_qk_norm* norm, const vm_hip_rope* rope, const int32_t* positions,
                           const int32_t* slots, void* q_out, void* stream) {
    clear_error();
    VM_TRY(check_kv_paged(cache, "kv_paged_append"));
    if (rows > 0 && !slots) return fail_inval("kv_paged_append: null pointer");
    AppendArgs a{};
    a.qkv = qkv;
    a.q_out = q_out;
    a.k_out = cache->k;
    a.v_out = cache->v;
    a.positions = positions;
    a.slots = slots;
    a.rows = rows;
    a.slot_count = cache->pages * cache->page_size;
    a.shift = log2_of(cache->page_size);
    return append("kv_paged_append", a, cache->dtype, heads, cache->kv_heads, cache->head_dim, norm, rope, stream);
}

int vm_hip_qk_norm_rope(const void* qkv, int dtype, int64_t rows, int64_t heads, int64_t kv_heads, int64_t head_dim,
                        const vm_hip_qk_norm* norm, const vm_hip_rope* rope, const int32_t* positions, void* q_out,
                        void* k_out, void* stream) {
    clear_error();
    if (!known_dtype(dtype)) return fail_inval("qk_norm_rope: dtype must be F32, F16 or BF16");
    if (head_dim != 64 && head_dim != 128) return fail_inval("qk_norm_rope: head_dim must be 64 or 128");
    if (kv_heads < 1 || kv_heads > 4096) return fail_inval("qk_norm_rope: kv_heads out of range");
    AppendArgs a{};
    a.qkv = qkv;
    a.q_out = q_out;
    a.k_out = k_out;
    a.positions = positions;
    a.rows = rows;
    a.slot_count = 1;
    return append("qk_norm_rope", a, dtype, heads, kv_heads, head_dim, norm, rope, stream);
}

}  // extern "C"
