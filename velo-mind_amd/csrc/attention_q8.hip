// Attention over the INT8 KV cache (kv_q8.hip) for one or many tokens of a
// sequence: decoded tokens, prompts and trees of drafted tokens.
//
//   o_r = sum_j p_rj sv_j cv_j / sum_j p_rj,   p_rj = exp(s_rj - max_j s_rj),
//   s_rj = scale sk_j (q_r . ck_j)
//
// with codes ck, cv and scales sk, sv of cache row j.  The query heads of a
// KV head read the same rows, so the (token, head) pairs of a KV head are its
// query rows, r = token G + head, and 16 of them fill an MFMA tile: a decoded
// token of a grouped model costs one tile and one pass over the cache.
//
// Codes are exact in fp16, so both products run on v_mfma_f32_16x16x32_f16:
// fp32 queries and weights as two fp16 parts (22 bits), 16-bit ones as one.
// A[i][k] and B[k][j] sit in lane i (j) + 16 (k / 8), element k % 8; D[i][j]
// in lane j + 16 (i / 4), element i % 4.  Both products are computed
// transposed, S^T = K Q^T and O^T = V^T P^T, so that query row lr = lane % 16
// owns its column of both: its statistics and factors need no shuffles.  The
// tiles' rows are numbered so that nothing has to move between them:
//   S^T  tile bt (0, 1) of a 32-key block has key 8 (i / 4) + 4 bt + i % 4 in
//        row i: lane group lg = lane / 16 then holds scores of keys 8 lg ..
//        + 7, the B operand P^T of the second product as it stands;
//   K    is read 16 bytes a lane, dims 64 h + 16 lg ..; the two k-steps of a
//        64-dim slab take its halves (the order of a sum's terms is free);
//   O^T  row i of tile db is dim (D / 16) i + db: a lane reads D / 16
//        adjacent codes of each of its eight keys and transposes them in
//        registers with byte permutes while it widens them.
// Widening: code ^ 0x80 behind the byte 0x64 is fp16 1152 + code, one packed
// subtraction away.
//
// Weights meet fp16 as p sv 2^(14 - E), 2^E above the largest sv seen: what
// the second part cannot hold is below 2^-39 of the largest.
//
// A workgroup of four waves takes 16 RW query rows and a share of the keys;
// its KS = 4 / RW key groups take turns at 32-key blocks, and their (max,
// sum, output) triples are merged through LDS.  Where few workgroups would
// leave the GPU idle the keys are split over several of them; each stores its
// triple in the workspace, and the one that draws the last ticket merges.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "kv_q8.h"
#include "vm_device.h"
#include "vm_internal.h"

namespace vmhip {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kBlock = 32;             // keys of a block
constexpr int kMaxSplits = 64;
constexpr int kMaxUnits = 1024;        // workgroup groups that split their keys
constexpr int64_t kTicketBytes = kMaxUnits * 4;
constexpr int kTargetGroups = 512;     // workgroups that fill 256 compute units twice

struct Args {
    const int8_t* kc;
    const float* ks;
    const int8_t* vc;
    const float* vs;
    const void* q;
    void* out;
    const int32_t* pos;
    const int32_t* counts;
    const uint64_t* tree;
    unsigned* tickets;
    char* parts;
    int batch, rows, heads, kv_heads, max_seq, words, splits, tiles;
    float scale;
};

// log2 of the power of two just above v (v >= 0 finite; 0 and subnormals: -126).
__device__ __forceinline__ int exponent_above(float v) { return static_cast<int>(__float_as_uint(v) >> 23) - 126; }

// Bytes 0, 1 (2, 3) of u = code ^ 0x80 as two fp16 codes.
__device__ __forceinline__ half2v widen_low(uint32_t u) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) -
           half2v{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
}
__device__ __forceinline__ half2v widen_high(uint32_t u) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) -
           half2v{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
}
__device__ __forceinline__ half8 join(half2v a, half2v b, half2v c, half2v d) {
    return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Maximum over the lanes of a row's four groups (lanes lr + 16 g).
__device__ __forceinline__ float max_groups(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float sum_groups(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

template <typename T>
__device__ __forceinline__ void load_query(const T* p, float (&x)[16]);
template <>
__device__ __forceinline__ void load_query<float>(const float* p, float (&x)[16]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const float4 v = reinterpret_cast<const float4*>(p)[u];
        x[4 * u] = v.x, x[4 * u + 1] = v.y, x[4 * u + 2] = v.z, x[4 * u + 3] = v.w;
    }
}
template <>
__device__ __forceinline__ void load_query<F16>(const F16* p, float (&x)[16]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const half8 v = reinterpret_cast<const half8*>(p)[u];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[8 * u + e] = static_cast<float>(v[e]);
    }
}
template <>
__device__ __forceinline__ void load_query<BF16>(const BF16* p, float (&x)[16]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const u32x4 v = reinterpret_cast<const u32x4*>(p)[u];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[8 * u + 2 * e] = __uint_as_float(v[e] << 16);
            x[8 * u + 2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ void store4(float* p, const float* y) { *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]); }
__device__ __forceinline__ void store4(F16* p, const float* y) {
    const half2v a{static_cast<_Float16>(y[0]), static_cast<_Float16>(y[1])};
    const half2v b{static_cast<_Float16>(y[2]), static_cast<_Float16>(y[3])};
    *reinterpret_cast<u32x2*>(p) = u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}
__device__ __forceinline__ void store4(BF16* p, const float* y) {
    *reinterpret_cast<u32x2*>(p) = u32x2{f32_to_bf16_ref(y[0]) | static_cast<uint32_t>(f32_to_bf16_ref(y[1])) << 16,
                                         f32_to_bf16_ref(y[2]) | static_cast<uint32_t>(f32_to_bf16_ref(y[3])) << 16};
}

// One workgroup's place: which rows, and which 32-key blocks of its keys.
// Both the kernel's waves and the last arrival's merge go by it.
template <int RW>
struct Place {
    int b, kh, tile, split, unit;
    int g, p0, n_tok, n_keys;   // group size, cached tokens, real tokens, cache rows that exist
    int active, first, last;    // workgroups that share the keys; this one's blocks
};

template <int RW>
__device__ __forceinline__ Place<RW> place(const Args& a) {
    Place<RW> w;
    int id = static_cast<int>(blockIdx.x);
    w.split = id % a.splits;
    id /= a.splits;
    w.unit = id;
    w.tile = id % a.tiles;
    id /= a.tiles;
    w.kh = id % a.kv_heads;
    w.b = id / a.kv_heads;
    w.g = a.heads / a.kv_heads;
    // (clamped where nothing changes: rows past max_seq, or all before row 0)
    w.p0 = max(min(a.pos[w.b], a.max_seq), -(1 << 21));
    w.n_tok = a.counts ? min(max(a.counts[w.b], 0), a.rows) : a.rows;
    const int64_t end = static_cast<int64_t>(w.p0) + w.n_tok;
    w.n_keys = static_cast<int>(min(max(end, int64_t(0)), static_cast<int64_t>(a.max_seq)));
    // A chain's tile sees the rows up to its last token's.
    int seen = w.n_keys;
    if (!a.tree) {
        const int t_last = min((w.tile * 16 * RW + 16 * RW - 1) / w.g, w.n_tok - 1);
        seen = static_cast<int>(min(static_cast<int64_t>(seen), max(static_cast<int64_t>(w.p0) + t_last + 1, int64_t(0))));
    }
    const int blocks = (seen + kBlock - 1) / kBlock;
    constexpr int kLeast = 2 * (4 / RW);   // blocks that are worth a workgroup
    const int share = max((blocks + a.splits - 1) / a.splits, kLeast);
    w.active = max((blocks + share - 1) / share, 1);
    w.first = w.split * share;
    w.last = min(blocks, w.first + share);
    return w;
}

template <typename T, int D, int RW>
__global__ __launch_bounds__(kThreads, 2) void attention_q8_kernel(const Args a) {
    constexpr int H = D / 64;              // 64-dim slabs
    constexpr int NC = D / 32;             // k-steps of a score
    constexpr int ND = D / 16;             // dim tiles; codes of a key that a lane reads
    constexpr int KS = 4 / RW;
    constexpr bool kTwo = sizeof(T) == 4;  // fp32 operands: two fp16 parts
    constexpr int NP = kTwo ? 2 : 1;
    __shared__ __align__(16) float scales_lds[4][2 * kBlock];
    __shared__ __align__(16) float merge_o[KS > 1 ? (KS - 1) * RW * 16 * D : 4];
    __shared__ float merge_ml[KS > 1 ? (KS - 1) * RW * 16 * 2 : 1];
    __shared__ unsigned ticket;

    const Place<RW> w = place<RW>(a);
    if (w.split >= w.active) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % RW, kg = wave / RW;
    const int lr = lane & 15, lg = lane >> 4;
    const int r = (w.tile * RW + wr) * 16 + lr;     // query row of this lane
    const int t = r / w.g, head = w.kh * w.g + r % w.g;
    const bool row_ok = t < w.n_tok;                // (rows past the last token's have t >= rows >= n_tok)
    const int t_first = (w.tile * RW + wr) * 16 / w.g;   // the wave's first token
    const bool wave_ok = t_first < w.n_tok;
    // Rows below `whole` are seen by every token of the wave.
    const int whole = min(a.tree ? w.p0 : w.p0 + t_first + 1, w.n_keys);

    // Q^T operand: Q[r][64 h + 16 lg + 8 s + j] in qf[.][2 h + s], scaled by the
    // power of two that puts the row's largest magnitude in [2^13, 2^14).
    half8 qf[NP][NC];
    float row_factor;
    {
        float x[H][16];
        const T* qp = static_cast<const T*>(a.q) +
                      ((static_cast<int64_t>(w.b) * a.heads + head) * a.rows + t) * D + 16 * lg;
        uint32_t m = 0;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (row_ok) {
                load_query(qp + 64 * h, x[h]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[h][e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) m = max(m, __float_as_uint(x[h][e]) & 0x7fffffffu);
        }
        m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16, 64)));
        m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32, 64)));
        const bool finite = m < 0x7f800000u;
        const int up = 14 - exponent_above(__uint_as_float(m));
        // exp2's argument: log2(e) times the score
        row_factor = finite ? ldexpf(a.scale * 1.44269504f, -up) : NAN;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = finite ? ldexpf(x[h][e], up) : 0.0f;
                const _Float16 hi = static_cast<_Float16>(v);
                qf[0][2 * h + e / 8][e % 8] = hi;
                if (kTwo) qf[NP - 1][2 * h + e / 8][e % 8] = static_cast<_Float16>(v - static_cast<float>(hi));
            }
    }

    const int64_t head_row = (static_cast<int64_t>(w.b) * a.kv_heads + w.kh) * a.max_seq;
    const uint32_t code_bytes = static_cast<uint32_t>(w.n_keys) * D;   // loads past it give zeros
    const __amdgpu_buffer_rsrc_t krs = buffer_rsrc(a.kc + head_row * D, code_bytes);
    const __amdgpu_buffer_rsrc_t vrs = buffer_rsrc(a.vc + head_row * D, code_bytes);
    const float* scale_src = (lane < kBlock ? a.ks : a.vs) + head_row;
    const uint32_t k_off = static_cast<uint32_t>(8 * (lr / 4) + lr % 4) * D + 16 * lg;
    const uint32_t v_off = static_cast<uint32_t>(8 * lg) * D + ND * lr;

    struct Codes {
        u32x4 k[2][H];
        uint32_t v[8][ND / 4];
        float s;
    };
    auto load = [&](int block, Codes& c) {
        const int k0 = block * kBlock;
        const uint32_t o = static_cast<uint32_t>(k0) * D;
        c.s = scale_src[min(k0 + (lane & (kBlock - 1)), w.n_keys - 1)];
#pragma unroll
        for (int bt = 0; bt < 2; ++bt)
#pragma unroll
            for (int h = 0; h < H; ++h) c.k[bt][h] = buffer_load16(krs, o + k_off + 4 * bt * D + 64 * h);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (ND == 8) {
                const u32x2 v = __builtin_bit_cast(
                    u32x2, __builtin_amdgcn_raw_buffer_load_b64(vrs, static_cast<int>(o + v_off + j * D), 0, 0));
                c.v[j][0] = v.x;
                c.v[j][1] = v.y;
            } else {
                c.v[j][0] = buffer_load4(vrs, o + v_off + j * D);
            }
        }
    };

    f32x4 acc[ND];   // O^T[dim ND (4 lg + e) + db][row lr] 2^(14 - v_exp)
#pragma unroll
    for (int db = 0; db < ND; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.0f;   // l: this lane's keys only
    int v_exp = -200;                        // E of the weights' unit

    auto compute = [&](int block, const Codes& c) {
        const int k0 = block * kBlock;
        float* sl = scales_lds[wave];
        sl[lane] = c.s;                       // keys' scales, then values'
        f32x4 st[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int bt = 0; bt < 2; ++bt) {
                    const uint32_t u0 = c.k[bt][h][2 * s] ^ 0x80808080u, u1 = c.k[bt][h][2 * s + 1] ^ 0x80808080u;
                    const half8 kf = join(widen_low(u0), widen_high(u0), widen_low(u1), widen_high(u1));
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        st[bt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[p][2 * h + s], st[bt], 0, 0, 0);
                }
        __builtin_amdgcn_wave_barrier();
        float sk[8], sv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sk[j] = sl[8 * lg + j];
            sv[j] = sl[kBlock + 8 * lg + j];
        }
        __builtin_amdgcn_wave_barrier();
        uint32_t sees = 0xffu;   // bit j: row lr sees key k0 + 8 lg + j
        const bool masked = k0 + kBlock > whole;
        if (masked) {
            const int key0 = k0 + 8 * lg;
            const int node0 = key0 - w.p0;   // of the call's own rows; negative: cached before
            if (a.tree) {
                const uint64_t* tw = a.tree + (static_cast<int64_t>(w.b) * a.rows + (row_ok ? t : 0)) * a.words;
                const int lo = max(node0, 0), wi = lo >> 6, sh = lo & 63;
                const uint64_t w0 = wi < a.words ? tw[wi] : 0, w1 = wi + 1 < a.words ? tw[wi + 1] : 0;
                const uint64_t win = sh ? w0 >> sh | w1 << (64 - sh) : w0;
                const int before = min(max(-node0, 0), 8);   // keys of the eight that were cached before
                sees = static_cast<uint32_t>(win) << before | ((1u << before) - 1);
            } else {
                const int n = t - node0 + 1;   // keys of the eight up to the token's own
                sees = n >= 8 ? 0xffu : n > 0 ? (1u << n) - 1 : 0u;
            }
            const int n = w.n_keys - key0;
            sees &= n >= 8 ? 0xffu : n > 0 ? (1u << n) - 1 : 0u;
            if (!row_ok) sees = 0;
        }
        float v[8];
        float mt = -INFINITY, top = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = st[j / 4][j % 4] * (sk[j] * row_factor);
            if (masked && !(sees >> j & 1)) v[j] = -INFINITY;
            mt = fmaxf(mt, v[j]);
            top = fmaxf(top, sv[j]);   // (NaN is skipped)
        }
        mt = max_groups(mt);
        top = max_groups(top);
        const float m_new = fmaxf(m_run, mt);
        const float m_ref = m_new == -INFINITY ? 0.0f : m_new;
        const int e_new = max(v_exp, exponent_above(top));
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_ref);
        const float fall = ldexpf(alpha, v_exp - e_new);
        float ls = 0.0f;
        half8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float p = __builtin_amdgcn_exp2f(v[j] - m_ref);
            ls += p;
            float x = p * ldexpf(sv[j], 14 - e_new);
            if (masked && !(sees >> j & 1)) x = 0.0f;   // (0 times a NaN scale)
            const _Float16 hi = static_cast<_Float16>(x);
            ph[j] = hi;
            if (kTwo) pl[j] = static_cast<_Float16>(x - static_cast<float>(hi));
        }
        l_run = fmaf(l_run, alpha, ls);
        m_run = m_new;
        v_exp = e_new;
        if (__any(fall != 1.0f)) {
#pragma unroll
            for (int db = 0; db < ND; ++db) acc[db] *= fall;
        }
        // V^T: four dim tiles from four adjacent codes of eight keys.
#pragma unroll
        for (int d4 = 0; d4 < ND / 4; ++d4) {
            half2v f[4][4];   // [dim tile][key pair]
#pragma unroll
            for (int jp = 0; jp < 4; ++jp) {
                const uint32_t u0 = c.v[2 * jp][d4] ^ 0x80808080u, u1 = c.v[2 * jp + 1][d4] ^ 0x80808080u;
                const uint32_t m01 = __builtin_amdgcn_perm(u1, u0, 0x05010400u);
                const uint32_t m23 = __builtin_amdgcn_perm(u1, u0, 0x07030602u);
                f[0][jp] = widen_low(m01);
                f[1][jp] = widen_high(m01);
                f[2][jp] = widen_low(m23);
                f[3][jp] = widen_high(m23);
            }
#pragma unroll
            for (int db = 0; db < 4; ++db) {
                const half8 vf = join(f[db][0], f[db][1], f[db][2], f[db][3]);
                acc[4 * d4 + db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, acc[4 * d4 + db], 0, 0, 0);
                if (kTwo) acc[4 * d4 + db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, acc[4 * d4 + db], 0, 0, 0);
            }
        }
    };

    if (wave_ok) {
        Codes c0, c1;
        int block = w.first + kg;
        if (block < w.last) {
            load(block, c0);
            while (true) {
                if (block + KS < w.last) load(block + KS, c1);
                compute(block, c0);
                block += KS;
                if (block >= w.last) break;
                if (block + KS < w.last) load(block + KS, c0);
                compute(block, c1);
                block += KS;
                if (block >= w.last) break;
            }
        }
    }
    l_run = sum_groups(l_run);
    float o[4][ND];   // dims ND (4 lg + e) + db of row lr
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int db = 0; db < ND; ++db) o[e][db] = ldexpf(acc[db][e], v_exp - 14);

    // Merge the key groups into group 0.
    if constexpr (KS > 1) {
        if (kg > 0) {
            float* d = merge_o + (((kg - 1) * RW + wr) * 16 + lr) * D + 4 * ND * lg;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int u = 0; u < ND / 4; ++u) store4(d + ND * e + 4 * u, &o[e][4 * u]);
            if (lg == 0) {
                merge_ml[(((kg - 1) * RW + wr) * 16 + lr) * 2] = m_run;
                merge_ml[(((kg - 1) * RW + wr) * 16 + lr) * 2 + 1] = l_run;
            }
        }
        __syncthreads();
        if (kg == 0) {
            float m = m_run;
#pragma unroll
            for (int k = 0; k < KS - 1; ++k) m = fmaxf(m, merge_ml[((k * RW + wr) * 16 + lr) * 2]);
            const float m_ref = m == -INFINITY ? 0.0f : m;
            const float f0 = __builtin_amdgcn_exp2f(m_run - m_ref);
            l_run *= f0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int db = 0; db < ND; ++db) o[e][db] *= f0;
#pragma unroll
            for (int k = 0; k < KS - 1; ++k) {
                const float* ml = merge_ml + ((k * RW + wr) * 16 + lr) * 2;
                const float f = __builtin_amdgcn_exp2f(ml[0] - m_ref);
                l_run = fmaf(ml[1], f, l_run);
                const float* s = merge_o + ((k * RW + wr) * 16 + lr) * D + 4 * ND * lg;
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int db = 0; db < ND; ++db) o[e][db] = fmaf(s[ND * e + db], f, o[e][db]);
            }
            m_run = m;
        }
    }
    if (w.active == 1) {
        if (kg == 0 && row_ok) {
            const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;   // (no row seen: zeros)
            T* d = static_cast<T*>(a.out) + ((static_cast<int64_t>(w.b) * a.rows + t) * a.heads + head) * D + 4 * ND * lg;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int u = 0; u < ND / 4; ++u) {
                    const float y[4] = {o[e][4 * u] * inv, o[e][4 * u + 1] * inv, o[e][4 * u + 2] * inv,
                                        o[e][4 * u + 3] * inv};
                    store4(d + ND * e + 4 * u, y);
                }
        }
        return;
    }
    // Several workgroups share the keys: [16 RW][D] outputs, then maxima and sums.
    constexpr uint32_t kPart = 16 * RW * (D + 2) * 4;
    char* unit_parts = a.parts + static_cast<int64_t>(w.unit) * a.splits * kPart;
    if (kg == 0) {
        const __amdgpu_buffer_rsrc_t prs = buffer_rsrc(unit_parts + static_cast<int64_t>(w.split) * kPart, kPart);
        const uint32_t at = static_cast<uint32_t>(wr * 16 + lr) * D * 4 + 16 * ND * lg;
        if (row_ok) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int u = 0; u < ND / 4; ++u)
                    coherent_store16(prs, at + 4 * ND * e + 16 * u,
                                     u32x4{__float_as_uint(o[e][4 * u]), __float_as_uint(o[e][4 * u + 1]),
                                           __float_as_uint(o[e][4 * u + 2]), __float_as_uint(o[e][4 * u + 3])});
        }
        if (lg == 0) {
            float* ml = reinterpret_cast<float*>(unit_parts + static_cast<int64_t>(w.split) * kPart) + 16 * RW * D;
            coherent_store(ml + wr * 16 + lr, m_run);
            coherent_store(ml + 16 * RW + wr * 16 + lr, l_run);
        }
        publish_partials();
    }
    __syncthreads();
    if (threadIdx.x == 0) ticket = ticket_take(a.tickets + w.unit, w.active);
    __syncthreads();
    if (ticket != static_cast<unsigned>(w.active - 1)) return;
    if (threadIdx.x == 0) __hip_atomic_store(a.tickets + w.unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // The last arrival: thread (row, 4 dims), workgroups in order.
    for (int item = threadIdx.x; item < 16 * RW * (D / 4); item += kThreads) {
        const int row = item / (D / 4), d4 = item % (D / 4);
        const int rr = w.tile * RW * 16 + row, tt = rr / w.g;
        if (tt >= w.n_tok) continue;
        float m = -INFINITY;
        for (int s = 0; s < w.active; ++s)
            m = fmaxf(m, coherent_load(reinterpret_cast<const float*>(unit_parts + static_cast<int64_t>(s) * kPart) +
                                       16 * RW * D + row));
        const float m_ref = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, y[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < w.active; ++s) {
            const char* part = unit_parts + static_cast<int64_t>(s) * kPart;
            const float* ml = reinterpret_cast<const float*>(part) + 16 * RW * D;
            const float f = __builtin_amdgcn_exp2f(coherent_load(ml + row) - m_ref);
            l = fmaf(coherent_load(ml + 16 * RW + row), f, l);
            const u32x4 x = coherent_load16(buffer_rsrc(part, kPart), static_cast<uint32_t>(item) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = fmaf(__uint_as_float(x[e]), f, y[e]);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= inv;
        store4(static_cast<T*>(a.out) +
                   ((static_cast<int64_t>(w.b) * a.rows + tt) * a.heads + w.kh * w.g + rr % w.g) * D + 4 * d4,
               y);
    }
}

// Row blocks of a workgroup, tiles, and workgroups that share a tile's keys.
struct Plan {
    int rw, splits;
    int64_t tiles, units;
    int64_t bytes;
};

Plan plan(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t d, int64_t max_seq) {
    Plan p;
    const int64_t r = rows * (heads / kv_heads);
    p.rw = r <= 16 ? 1 : r <= 32 ? 2 : 4;
    p.tiles = (r + 16 * p.rw - 1) / (16 * p.rw);
    p.units = batch * kv_heads * p.tiles;
    const int64_t most = (max_seq + kBlock * 2 * (4 / p.rw) - 1) / (kBlock * 2 * (4 / p.rw));
    int64_t s = p.units > 0 && p.units < kTargetGroups ? (kTargetGroups + p.units - 1) / p.units : 1;
    s = std::min<int64_t>(std::min<int64_t>(s, kMaxSplits), most);
    p.splits = static_cast<int>(std::max<int64_t>(s, 1));
    p.bytes = p.splits > 1 ? kTicketBytes + p.units * p.splits * (16 * p.rw * (d + 2) * 4) : 0;
    return p;
}

int check_shape(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t d, int64_t max_seq) {
    if (d != 64 && d != 128) return fail_inval("attention_q8: head_dim must be 64 or 128");
    if (batch < 0 || batch > 65535 || kv_heads < 1 || kv_heads > 4096 || max_seq < 1 || max_seq > 0x7fffffff / d)
        return fail_inval("attention_q8: batch, kv_heads or max_seq out of range");
    if (rows < 0 || rows > (1 << 20) || heads < 1 || heads > 65536 || heads % kv_heads ||
        rows * (heads / kv_heads) > (1 << 30))
        return fail_inval("attention_q8: bad rows or heads");
    if (batch && rows && plan(batch, rows, heads, kv_heads, d, max_seq).units > (1 << 30))
        return fail_inval("attention_q8: too many rows for one call");
    return 0;
}

template <typename T, int D, int RW>
void launch(const Args& a, int64_t grid, hipStream_t stream) {
    hipLaunchKernelGGL((attention_q8_kernel<T, D, RW>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, a);
}

template <typename T, int D>
void launch_rows(const Args& a, int rw, int64_t grid, hipStream_t stream) {
    if (rw == 1)
        launch<T, D, 1>(a, grid, stream);
    else if (rw == 2)
        launch<T, D, 2>(a, grid, stream);
    else
        launch<T, D, 4>(a, grid, stream);
}

}  // namespace
}  // namespace vmhip

using namespace vmhip;

extern "C" {

int64_t vm_hip_attention_q8_workspace_bytes(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                            int64_t head_dim, int64_t max_seq) {
    clear_error();
    VM_TRY(check_shape(batch, rows, heads, kv_heads, head_dim, max_seq));
    if (batch == 0 || rows == 0) return 0;
    return plan(batch, rows, heads, kv_heads, head_dim, max_seq).bytes;
}

int vm_hip_attention_q8(const vm_hip_kv_q8* cache, const void* q, void* out, int dtype, int64_t rows, int64_t heads,
                        const int32_t* pos, const int32_t* counts, const uint64_t* tree, float scale, void* workspace,
                        int64_t workspace_bytes, void* stream) {
    clear_error();
    VM_TRY(check_kv_q8(cache, "attention_q8"));
    VM_TRY(check_shape(cache->batch, rows, heads, cache->kv_heads, cache->head_dim, cache->max_seq));
    if (dtype != VM_HIP_DTYPE_F32 && dtype != VM_HIP_DTYPE_F16 && dtype != VM_HIP_DTYPE_BF16)
        return fail_inval("attention_q8: dtype must be F32, F16 or BF16");
    if (rows == 0 || cache->batch == 0) return 0;
    if (!q || !out || !pos) return fail_inval("attention_q8: null pointer");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
        return fail_inval("attention_q8: q and out must be 16-byte aligned");
    if (!(scale < INFINITY)) return fail_inval("attention_q8: scale must be finite");
    const Plan p = plan(cache->batch, rows, heads, cache->kv_heads, cache->head_dim, cache->max_seq);
    if (p.bytes > 0 &&
        (!workspace || workspace_bytes < p.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))
        return fail_inval("attention_q8: workspace smaller than vm_hip_attention_q8_workspace_bytes or unaligned");
    Args a;
    a.kc = cache->k_codes;
    a.ks = cache->k_scales;
    a.vc = cache->v_codes;
    a.vs = cache->v_scales;
    a.q = q;
    a.out = out;
    a.pos = pos;
    a.counts = counts;
    a.tree = tree;
    a.tickets = static_cast<unsigned*>(workspace);
    a.parts = static_cast<char*>(workspace) + (p.bytes > 0 ? kTicketBytes : 0);
    a.batch = static_cast<int>(cache->batch);
    a.rows = static_cast<int>(rows);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(cache->kv_heads);
    a.max_seq = static_cast<int>(cache->max_seq);
    a.words = static_cast<int>((rows + 63) / 64);
    a.splits = p.splits;
    a.tiles = static_cast<int>(p.tiles);
    a.scale = scale > 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(cache->head_dim));
    const int64_t grid = p.units * p.splits;
    auto s = static_cast<hipStream_t>(stream);
    const bool wide = cache->head_dim == 128;
    if (dtype == VM_HIP_DTYPE_F32)
        wide ? launch_rows<float, 128>(a, p.rw, grid, s) : launch_rows<float, 64>(a, p.rw, grid, s);
    else if (dtype == VM_HIP_DTYPE_F16)
        wide ? launch_rows<F16, 128>(a, p.rw, grid, s) : launch_rows<F16, 64>(a, p.rw, grid, s);
    else
        wide ? launch_rows<BF16, 128>(a, p.rw, grid, s) : launch_rows<BF16, 64>(a, p.rw, grid, s);
    return check_launch("attention_q8", s);
}

}  // extern "C"
