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
// Weights meet fp16 as p sv 2^(8 - E + u), p below 2^7: 2^E is above the scales of
// the values that the wave's rows have seen, and u is a row's own.  While all
// scales that a row may have taken its reference from are 2^(E - 5) at least (and
// none is that of zeros, 1), u is 0, and the wave keeps nothing for it.  From then
// on (`wide`) a row's largest p sv is known, of keys that it sees and that hold
// more than zeros, and u puts it near 2^8.  What fp16 (its second part, of fp32
// calls) cannot hold is below 2^-28 of the row's largest p sv either way, whatever
// the other rows see.  (With one unit for all a wave's rows, from all its keys,
// values were lost beside rows of zeros and beside large values that a row does
// not see; the units cost 2 us of 58 for 1000 rows behind 3001; with rows of zeros in
// the cache, which every block is then searched for, that call takes 63 to 68 us,
// a tree of 24 over 131000 215 to 217.)
//
// A workgroup of four waves takes 16 RT query rows and a share of the keys;
// its waves take turns at 32-key blocks, the next block's codes in registers
// while one is computed, and their (reference, sum, output) triples are merged
// through LDS.  Where few workgroups would leave the GPU idle the keys are
// split over several of them; each stores its triple in the workspace, and the
// one that draws the last ticket merges.
//
// MI355X, passes back to back: 32 tokens over ragged caches of up to 8000, 64
// heads of 128, bf16: 88 us, 4.6 TB/s of codes and scales (HBM: a large copy
// reaches 4.8 to 5.4); 1000 rows of 32 heads of 64 behind 3001 cached, f16: 58 us,
// 490 TFLOP/s, f32: 90 us; 24 nodes of 64 heads of 128 over 131000, bf16: 194 us,
// 530 TFLOP/s (VALU: widening and softmax, ten to twelve instructions beside an
// MFMA, the matrix cores busy 17 to 20 % of the cycles); one token of 32 heads over
// 2000: 7.6 us, 16 nodes: 8.2 (the chain position - codes - LDS merge - ticket -
// join).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

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
constexpr int kWaves = kThreads / 64;
constexpr int kBlock = 32;             // keys of a block
constexpr int kLeast = 2 * kWaves;     // blocks that are worth a workgroup
constexpr int kMaxSplits = 64;
constexpr int kMaxUnits = 512;         // workgroup groups that split their keys
constexpr int kTicketStride = 16;      // a ticket has a 64-byte line of its own
constexpr int64_t kTicketBytes = kMaxUnits * kTicketStride * 4;
constexpr int kTargetGroups = 512;     // workgroups that fill 256 compute units twice
static_assert(kTargetGroups <= kMaxUnits, "calls of more units do not split");

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
__device__ __forceinline__ half2v widen_bits(uint32_t bits) {
    return __builtin_bit_cast(half2v, bits) - half2v{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
}
__device__ __forceinline__ half2v widen_low(uint32_t u) {
    return widen_bits(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
}
__device__ __forceinline__ half2v widen_high(uint32_t u) {
    return widen_bits(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
}
__device__ __forceinline__ half8 join(half2v a, half2v b, half2v c, half2v d) {
    return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Bits of the 16 lanes lr of a lane's group joined.
__device__ __forceinline__ uint32_t join_rows(uint32_t v) {
    int x = static_cast<int>(v);
    x |= __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false);   // row_ror:1
    x |= __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false);
    x |= __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false);
    x |= __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false);
    return static_cast<uint32_t>(x);
}

// Maximum and sum over the lanes of a row's four groups (lanes lr + 16 g).
__device__ __forceinline__ float max_groups(float v) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    unsigned q[2];
    __builtin_memcpy(q, &p, sizeof q);
    v = fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    __builtin_memcpy(q, &h, sizeof q);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
    v = swap_rows_add(v, v);
    return swap_halves_add(v, v);
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
struct Place {
    int b, kh, tile, split, unit;
    int g, p0, n_tok, n_keys;   // group size, cached tokens, real tokens, cache rows that exist
    int active, first, last;    // workgroups that share the keys; this one's blocks
};

// Workgroups go to the XCDs in turn.  The tiles of a (sequence, head, share of
// the keys) read the same codes, so where the count of those allows they are
// placed on one XCD, next to each other, the tiles that see the most keys
// first; else they are as far apart as the others are many.
template <int RT>
__device__ __forceinline__ Place place(const Args& a) {
    Place w;
    int id = static_cast<int>(blockIdx.x);
    const int shares = a.batch * a.kv_heads * a.splits;
    int share;
    if (shares % 8 == 0) {
        const int j = id / 8;
        w.tile = a.tiles - 1 - j % a.tiles;
        share = j / a.tiles * 8 + id % 8;
    } else {
        w.tile = a.tiles - 1 - id / shares;
        share = id % shares;
    }
    w.split = share % a.splits;
    share /= a.splits;
    w.unit = share * a.tiles + w.tile;
    w.kh = share % a.kv_heads;
    w.b = share / a.kv_heads;
    w.g = a.heads / a.kv_heads;
    // (clamped where nothing changes: rows past max_seq, or all before row 0)
    w.p0 = max(min(a.pos[w.b], a.max_seq), -(1 << 21));
    w.n_tok = a.counts ? min(max(a.counts[w.b], 0), a.rows) : a.rows;
    w.n_keys = min(max(w.p0 + w.n_tok, 0), a.max_seq);
    // A chain's tile sees the rows up to its last token's.
    int seen = w.n_keys;
    if (!a.tree) seen = min(seen, max(w.p0 + min((w.tile * 16 * RT + 16 * RT - 1) / w.g, w.n_tok - 1) + 1, 0));
    const int blocks = (seen + kBlock - 1) / kBlock;
    const int each = max((blocks + a.splits - 1) / a.splits, kLeast);
    w.active = max((blocks + each - 1) / each, 1);
    w.first = w.split * each;
    w.last = min(blocks, w.first + each);
    return w;
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(kThreads, 2) void attention_q8_kernel(const Args a) {
    constexpr int H = D / 64;              // 64-dim slabs
    constexpr int NC = D / 32;             // k-steps of a score
    constexpr int ND = D / 16;             // dim tiles; codes of a key that a lane reads
    constexpr bool kTwo = sizeof(T) == 4;  // fp32 operands: two fp16 parts
    constexpr int NP = kTwo ? 2 : 1;
    constexpr int kRows = 16 * RT;
    // A weight may exceed 1 by this much (log2) before its row's reference moves:
    // with one unit some row of a wave moved in most blocks.
    constexpr float kHeadroom = 7.0f;
    constexpr int kUnit = 8;               // weights in units of 2^(E - kUnit - u): below 2^15
    constexpr int kNear = 4;               // scales from 2^(E - 5) up need no u
    constexpr float kUnset = -3e38f;       // limit of a row that has a reference and no weight yet
    __shared__ __align__(16) float scales_lds[kWaves][2 * kBlock];
    __shared__ __align__(16) float merge_o[kWaves][kRows * D];
    __shared__ float merge_m[kWaves][kRows], merge_l[kWaves][kRows];
    __shared__ unsigned ticket;

    const Place w = place<RT>(a);
    if (w.split >= w.active) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, lg = lane >> 4;
    const int r0 = w.tile * kRows;                  // the tile's first row, (token, head of the group)
    const int t_first = r0 / w.g;
    if (t_first >= w.n_tok) return;                 // padding only
    // Rows below `whole` are seen by every token of the tile.
    const int whole = min(a.tree ? w.p0 : w.p0 + t_first + 1, w.n_keys);

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

    // The first block's codes are on their way while the queries are prepared.
    Codes c0, c1;
    int block = w.first + wave;
    if (block < w.last) load(block, c0);

    // Q^T operands: Q[row][64 h + 16 lg + 8 s + j] in qf[.][.][2 h + s], scaled by
    // the power of two that puts the row's largest magnitude in [2^13, 2^14).
    half8 qf[RT][NP][NC];
    float row_factor[RT];   // of a score's log2
    int token[RT];          // -1: no row
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = r0 + 16 * rt + lr, t = r / w.g;
        const bool row_ok = t < w.n_tok;
        token[rt] = row_ok ? t : -1;
        float x[H][16];
        const T* qp = static_cast<const T*>(a.q) +
                      ((static_cast<int64_t>(w.b) * a.heads + w.kh * w.g + r % w.g) * a.rows + t) * D + 16 * lg;
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
        row_factor[rt] = finite ? ldexpf(a.scale * 1.44269504f, -up) : NAN;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = finite ? ldexpf(x[h][e], up) : 0.0f;
                const _Float16 hi = static_cast<_Float16>(v);
                qf[rt][0][2 * h + e / 8][e % 8] = hi;
                if (kTwo) qf[rt][NP - 1][2 * h + e / 8][e % 8] = static_cast<_Float16>(v - static_cast<float>(hi));
            }
    }

    f32x4 acc[RT][ND];   // O^T[dim ND (4 lg + e) + db][row lr] 2^(kUnit - v_exp + u)
    float m_run[RT];     // the score (less the row's factor) that weighs 1
    float limit[RT];     // how far a score may pass it (log2); -inf before the first key
    float l_run[RT];     // sum of this lane's keys' weights
    // Of a row, where scales lie far apart (`wide`); in LDS until the merge needs the place:
    float* e_run = merge_m[wave] + lr;   // [16 rt] log2 of the row's largest p sv; -inf: none
    float* unit = merge_l[wave] + lr;    // [16 rt] 2^u
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int db = 0; db < ND; ++db) acc[rt][db] = f32x4{0.f, 0.f, 0.f, 0.f};
        m_run[rt] = l_run[rt] = 0.0f;
        limit[rt] = -INFINITY;
    }
    int v_exp = -200;       // E
    int lowest = 200;       // the smallest scales (log2) of blocks in which a reference moved
    bool wide = false;      // scales lie far apart, or there may be rows of zeros
    bool shifted = false;   // some row of the wave has another u than 0

    // kMasked: some row does not see the whole block (or the block ends past the
    // cache).  Two copies of the code: the masks cost a quarter of a block's time.
    auto compute = [&](auto masked_tag, int block, const Codes& c) {
        constexpr bool kMasked = decltype(masked_tag)::value;
        const int k0 = block * kBlock;
        float* sl = scales_lds[wave];
        sl[lane] = c.s;                       // keys' scales, then values'
        f32x4 st[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) st[rt][0] = st[rt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int bt = 0; bt < 2; ++bt) {
                    const uint32_t u0 = c.k[bt][h][2 * s] ^ 0x80808080u, u1 = c.k[bt][h][2 * s + 1] ^ 0x80808080u;
                    const half8 kf = join(widen_low(u0), widen_high(u0), widen_low(u1), widen_high(u1));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int p = 0; p < NP; ++p)
                            st[rt][bt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][p][2 * h + s], st[rt][bt], 0, 0, 0);
                }
        __builtin_amdgcn_wave_barrier();
        float sk[8], sv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sk[j] = sl[8 * lg + j];
            sv[j] = sl[kBlock + 8 * lg + j];
        }
        __builtin_amdgcn_wave_barrier();
        // Keys of zeros count for nothing.
        const auto drop_zeros = [&]() {
            uint32_t holds = 0;   // bit j: key 8 lg + j has another code than 0
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t bits = c.v[j][0];
#pragma unroll
                for (int u = 1; u < ND / 4; ++u) bits |= c.v[j][u];
                holds |= bits ? 1u << j : 0u;
            }
            holds = join_rows(holds);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(holds >> j & 1) && sv[j] == sv[j]) sv[j] = 0.0f;
        };
        if (wide) drop_zeros();
        // Scores less the row's reference (and its factor), and whether that or
        // the weights' unit has to move: rarely, after the first blocks.
        uint32_t sees[RT];   // bit j: the row sees key k0 + 8 lg + j
        float mt[RT];
        float top = fabsf(sv[0]);   // (NaN is skipped)
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, fabsf(sv[j]));
        bool moves = top == top && exponent_above(top) > v_exp;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            sees[rt] = 0xffu;
            if (kMasked) {
                const int key0 = k0 + 8 * lg;
                const int node0 = key0 - w.p0;   // of the call's own rows; negative: cached before
                if (a.tree) {
                    const uint64_t* tw = a.tree + (static_cast<int64_t>(w.b) * a.rows + max(token[rt], 0)) * a.words;
                    const int lo = max(node0, 0), wi = lo >> 6, sh = lo & 63;
                    const uint64_t w0 = wi < a.words ? tw[wi] : 0, w1 = wi + 1 < a.words ? tw[wi + 1] : 0;
                    const uint64_t win = sh ? w0 >> sh | w1 << (64 - sh) : w0;
                    const int before = min(max(-node0, 0), 8);   // keys of the eight that were cached before
                    sees[rt] = static_cast<uint32_t>(win) << before | ((1u << before) - 1);
                } else {
                    const int n = token[rt] - node0 + 1;   // keys of the eight up to the token's own
                    sees[rt] = n >= 8 ? 0xffu : n > 0 ? (1u << n) - 1 : 0u;
                }
                const int n = w.n_keys - key0;
                sees[rt] &= n >= 8 ? 0xffu : n > 0 ? (1u << n) - 1 : 0u;
                if (token[rt] < 0) sees[rt] = 0;
            }
            mt[rt] = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float v = fmaf(st[rt][j / 4][j % 4], sk[j], -m_run[rt]);
                if (kMasked && !(sees[rt] >> j & 1)) v = -INFINITY;
                st[rt][j / 4][j % 4] = v;
                mt[rt] = fmaxf(mt[rt], v);
            }
            moves = moves || mt[rt] * row_factor[rt] > limit[rt];
        }
        if (__any(moves)) {
            uint32_t seen_by = 0xffu;   // keys that some row of the wave sees
            if (kMasked) {
                seen_by = sees[0];
#pragma unroll
                for (int rt = 1; rt < RT; ++rt) seen_by |= sees[rt];
                seen_by = join_rows(seen_by);
            }
            const auto above_all = [&]() {   // E with this block's keys
                float most = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!kMasked || (seen_by >> j & 1)) most = fmaxf(most, fabsf(sv[j]));
                return __builtin_amdgcn_readfirstlane(max(v_exp, exponent_above(max_groups(most))));
            };
            int e_new = above_all();
            if (!wide) {
                float least = INFINITY;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!kMasked || (seen_by >> j & 1)) least = fminf(least, fabsf(sv[j]));
                lowest = __builtin_amdgcn_readfirstlane(min(lowest, exponent_above(-max_groups(-least))));
                bool one = false;   // (the scale of a row of zeros)
                if (e_new >= 1 && e_new <= 1 + kNear) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) one |= sv[j] == 1.0f;
                }
                if (lowest < e_new - kNear || __any(one)) {
                    wide = true;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        e_run[16 * rt] = limit[rt] == -INFINITY ? -INFINITY : static_cast<float>(v_exp - kNear);
                        unit[16 * rt] = 1.0f;
                    }
                }
            }
            if (wide) {
                drop_zeros();
                e_new = above_all();
            }
            const int drop = e_new - v_exp;
            v_exp = e_new;
            bool any_unit = false;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float most = max_groups(mt[rt]);
                const bool first = limit[rt] == -INFINITY;
                const bool seen = most > -INFINITY && row_factor[rt] == row_factor[rt];
                const float up = !seen ? 0.0f : first ? most : fmaxf(most, 0.0f);
                m_run[rt] += up;
                const float fall = first ? 1.0f : __builtin_amdgcn_exp2f(-up * row_factor[rt]);
                if (seen) limit[rt] = kHeadroom;
                l_run[rt] *= fall;
#pragma unroll
                for (int j = 0; j < 8; ++j) st[rt][j / 4][j % 4] -= up;
                int more = -drop;   // log2 of what the row's outputs grow by for their units
                if (wide) {
                    float w = -INFINITY;   // log2 of the row's largest p sv of this block
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (!kMasked || (sees[rt] >> j & 1))
                            w = fmaxf(w, fmaf(st[rt][j / 4][j % 4], row_factor[rt], __builtin_amdgcn_logf(fabsf(sv[j]))));
                    float e = e_run[16 * rt];
                    if (seen) e = fmaxf(e - up * row_factor[rt], max_groups(w));
                    e_run[16 * rt] = e;
                    const bool none = e == -INFINITY;
                    e += static_cast<float>(kUnit - v_exp);
                    const int u = none || (e >= kUnit - kNear && e <= kUnit + kNear) ? 0 : kUnit - static_cast<int>(ceilf(fmaxf(e, -100.0f)));
                    more += u + 1 - exponent_above(unit[16 * rt]);
                    unit[16 * rt] = ldexpf(1.0f, u);
                    any_unit |= u != 0;
                    if (limit[rt] > -INFINITY) limit[rt] = none ? kUnset : kHeadroom - static_cast<float>(max(u, 0));
                }
                const float scaled = ldexpf(fall, more);
#pragma unroll
                for (int db = 0; db < ND; ++db) acc[rt][db] *= scaled;
            }
            shifted = __any(any_unit);
        }
        float su[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) su[j] = ldexpf(sv[j], kUnit - v_exp);
        half8 pf[RT][NP];
        const auto weigh = [&](auto shifted_tag) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float row_unit = decltype(shifted_tag)::value ? unit[16 * rt] : 1.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float p = __builtin_amdgcn_exp2f(st[rt][j / 4][j % 4] * row_factor[rt]);
                    float x = decltype(shifted_tag)::value ? p * row_unit * su[j] : p * su[j];
                    if (kMasked && !(sees[rt] >> j & 1)) p = x = 0.0f;   // (whatever the factor and the scale are)
                    l_run[rt] += p;
                    // 16-bit calls: one part, 2^-12 of the weight, as fp16 outputs are
                    // rounded (another part would double the second product's MFMAs).
                    // (Both parts have to come from one rounding of x: folded into its
                    // product, the first part's conversion would round another value.)
                    if (kTwo) asm("" : "+v"(x));
                    const _Float16 hi = static_cast<_Float16>(x);
                    pf[rt][0][j] = hi;
                    if (kTwo) pf[rt][NP - 1][j] = static_cast<_Float16>(x - static_cast<float>(hi));
                }
            }
        };
        if (shifted)
            weigh(std::true_type{});
        else
            weigh(std::false_type{});
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
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        acc[rt][4 * d4 + db] =
                            __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rt][p], acc[rt][4 * d4 + db], 0, 0, 0);
            }
        }
    };

    // A wave's blocks, the next one's codes on their way while one is computed;
    // the blocks that need masks come last.
    {
        while (block < w.last && (block + 1) * kBlock <= whole) {
            if (block + kWaves < w.last) load(block + kWaves, c1);
            compute(std::false_type{}, block, c0);
            block += kWaves;
            if (block >= w.last || (block + 1) * kBlock > whole) {
                c0 = c1;
                break;
            }
            if (block + kWaves < w.last) load(block + kWaves, c0);
            compute(std::false_type{}, block, c1);
            block += kWaves;
        }
        for (; block < w.last; block += kWaves) {
            if (block + kWaves < w.last) load(block + kWaves, c1);
            compute(std::true_type{}, block, c0);
            c0 = c1;
        }
    }
    // Every wave's triple to LDS (outputs without their unit); then thread
    // (row, four dims) merges the four.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float l = sum_groups(l_run[rt]);
        const int back = v_exp - kUnit + (wide ? 1 - exponent_above(unit[16 * rt]) : 0);
        float* d = merge_o[wave] + (16 * rt + lr) * D + 4 * ND * lg;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int u = 0; u < ND / 4; ++u) {
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = ldexpf(acc[rt][4 * u + i][e], back);
                store4(d + ND * e + 4 * u, y);
            }
        if (lg == 0) {
            merge_m[wave][16 * rt + lr] = limit[rt] == -INFINITY ? -INFINITY : m_run[rt] * row_factor[rt];
            merge_l[wave][16 * rt + lr] = l;
        }
    }
    __syncthreads();
    constexpr int kItems = kRows * D / 4 / kThreads;   // of a thread
    constexpr uint32_t kPart = kRows * (D + 2) * 4;
    char* unit_parts = a.parts + static_cast<int64_t>(w.unit) * a.splits * kPart;
    const __amdgpu_buffer_rsrc_t prs = buffer_rsrc(unit_parts, kPart * static_cast<uint32_t>(a.splits));
    const auto put = [&](int row, int d4, const float* y, float l) {
        const int r = r0 + row, t = r / w.g;
        if (t >= w.n_tok) return;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // (no row seen: zeros)
        const float z[4] = {y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv};
        store4(static_cast<T*>(a.out) +
                   ((static_cast<int64_t>(w.b) * a.rows + t) * a.heads + w.kh * w.g + r % w.g) * D + 4 * d4,
               z);
    };
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int item = i * kThreads + threadIdx.x, row = item / (D / 4), d4 = item % (D / 4);
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
        if (w.active == 1) {
            put(row, d4, y, l);
            continue;
        }
        // Several workgroups share the keys: [rows][D] outputs, then maxima and sums.
        const uint32_t part = static_cast<uint32_t>(w.split) * kPart;
        coherent_store16(prs, part + static_cast<uint32_t>(item) * 16,
                         u32x4{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])});
        if (d4 == 0) {
            float* ml = reinterpret_cast<float*>(unit_parts + part) + kRows * D;
            coherent_store(ml + row, m);
            coherent_store(ml + kRows + row, l);
        }
    }
    if (w.active == 1) return;
    publish_partials();
    __syncthreads();
    if (threadIdx.x == 0) ticket = ticket_take(a.tickets + w.unit * kTicketStride, w.active);
    __syncthreads();
    if (ticket != static_cast<unsigned>(w.active - 1)) return;
    if (threadIdx.x == 0) __hip_atomic_store(a.tickets + w.unit * kTicketStride, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // The last arrival merges: the factor of every (workgroup, row) first, in
    // LDS, then thread (row, four dims) adds the workgroups in order, eight
    // loads in flight.
    constexpr int kFirst = kItems <= 2 ? 8 : 0;   // workgroups whose outputs are requested before the factors
    u32x4 early[kItems][kFirst + 1];
#pragma unroll
    for (int i = 0; i < kItems; ++i)
#pragma unroll
        for (int u = 0; u < kFirst; ++u)
            early[i][u] = u < w.active ? coherent_load16(prs, static_cast<uint32_t>(u) * kPart +
                                                                  (i * kThreads + threadIdx.x) * 16)
                                       : u32x4{0, 0, 0, 0};
    float* factor = merge_o[0];   // [active][rows]: at most 64 x 16 RT floats
    float* total = merge_m[0];
    static_assert(kMaxSplits * kRows <= kWaves * kRows * D, "factors fit");
    for (int row = threadIdx.x / 16; row < kRows; row += kThreads / 16) {
        const int s0 = threadIdx.x % 16;
        float mv[kMaxSplits / 16], lv[kMaxSplits / 16], m = -INFINITY;
#pragma unroll
        for (int u = 0; u < kMaxSplits / 16; ++u) {
            const int s = s0 + 16 * u;
            const float* ml = reinterpret_cast<const float*>(unit_parts + static_cast<int64_t>(s) * kPart) + kRows * D + row;
            mv[u] = s < w.active ? coherent_load(ml) : -INFINITY;
            lv[u] = s < w.active ? coherent_load(ml + kRows) : 0.0f;
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
            l = fmaf(lv[u], f, l);
            if (s < w.active) factor[s * kRows + row] = f;
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) l += __shfl_xor(l, o, 64);
        if (s0 == 0) total[row] = l;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int item = i * kThreads + threadIdx.x, row = item / (D / 4), d4 = item % (D / 4);
        float y[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < w.active; s0 += 8) {
            u32x4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                x[u] = s0 < kFirst ? early[i][kFirst ? u : 0] : s0 + u < w.active ? coherent_load16(prs, static_cast<uint32_t>(s0 + u) * kPart + item * 16)
                                         : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float f = s0 + u < w.active ? factor[(s0 + u) * kRows + row] : 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = fmaf(__uint_as_float(x[u][e]), f, y[e]);
            }
        }
        put(row, d4, y, total[row]);
    }
}

// 16-row tiles of a wave, row tiles, and workgroups that share a tile's keys.
struct Plan {
    int rt, splits;
    int64_t tiles, units;
    int64_t bytes;
};

Plan plan(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t d, int64_t max_seq, bool two) {
    Plan p;
    const int64_t r = rows * (heads / kv_heads);
    const int64_t most = (max_seq + kBlock * kLeast - 1) / (kBlock * kLeast);
    // More tiles a wave share the codes' widening, as far as registers go (fp32,
    // 64 dims: four spill; 16-bit, 128 dims, one wave per SIMD instead of two: 340
    // us against 201 for 24 tokens of 64 heads over 131000 keys; one tile: 303);
    // fewer where the keys cannot be shared out to enough workgroups (16 tokens
    // of 32 heads over 2000 keys: 9.0 us with one, 12.0 with two or four).
    p.rt = d == 64 && !two ? 4 : 2;
    while (p.rt > 1 && (r <= 8 * p.rt ||
                        batch * kv_heads * ((r + 16 * p.rt - 1) / (16 * p.rt)) * std::min<int64_t>(most, kMaxSplits) < kTargetGroups))
        p.rt /= 2;
    p.tiles = (r + 16 * p.rt - 1) / (16 * p.rt);
    p.units = batch * kv_heads * p.tiles;
    int64_t s = p.units > 0 && p.units < kTargetGroups ? kTargetGroups / p.units : 1;
    s = std::min<int64_t>(std::min<int64_t>(s, kMaxSplits), most);
    p.splits = static_cast<int>(std::max<int64_t>(s, 1));
    p.bytes = p.splits > 1 ? kTicketBytes + p.units * p.splits * (16 * p.rt * (d + 2) * 4) : 0;
    return p;
}

int check_shape(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t d, int64_t max_seq) {
    if (d != 64 && d != 128) return fail_inval("attention_q8: head_dim must be 64 or 128");
    if (batch < 0 || batch > 65535 || kv_heads < 1 || kv_heads > 4096 || max_seq < 1 || max_seq > 0x7fffffff / d)
        return fail_inval("attention_q8: batch, kv_heads or max_seq out of range");
    if (rows < 0 || rows > (1 << 20) || heads < 1 || heads > 65536 || heads % kv_heads ||
        rows * (heads / kv_heads) > (1 << 30))
        return fail_inval("attention_q8: bad rows or heads");
    // (a launch has less than 2^32 threads)
    if (batch && rows && plan(batch, rows, heads, kv_heads, d, max_seq, true).units >= (1 << 24))
        return fail_inval("attention_q8: too many rows for one call");
    return 0;
}

template <typename T, int D, int RT>
void launch(const Args& a, int64_t grid, hipStream_t stream) {
    hipLaunchKernelGGL((attention_q8_kernel<T, D, RT>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, a);
}

template <typename T>
void launch_rows(const Args& a, int64_t d, int rt, int64_t grid, hipStream_t stream) {
    if (d == 128)
        rt == 1 ? launch<T, 128, 1>(a, grid, stream) : launch<T, 128, 2>(a, grid, stream);
    else if (rt == 1)
        launch<T, 64, 1>(a, grid, stream);
    else if (rt == 2)
        launch<T, 64, 2>(a, grid, stream);
    else if constexpr (sizeof(T) == 2)   // (plan() gives fp32 two tiles at most)
        launch<T, 64, 4>(a, grid, stream);
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
    return std::max(plan(batch, rows, heads, kv_heads, head_dim, max_seq, false).bytes,
                    plan(batch, rows, heads, kv_heads, head_dim, max_seq, true).bytes);
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
    const Plan p = plan(cache->batch, rows, heads, cache->kv_heads, cache->head_dim, cache->max_seq,
                        dtype == VM_HIP_DTYPE_F32);
    const int64_t need = vm_hip_attention_q8_workspace_bytes(cache->batch, rows, heads, cache->kv_heads, cache->head_dim,
                                                             cache->max_seq);
    if (need > 0 &&
        (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))
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
    if (dtype == VM_HIP_DTYPE_F32)
        launch_rows<float>(a, cache->head_dim, p.rt, grid, s);
    else if (dtype == VM_HIP_DTYPE_F16)
        launch_rows<F16>(a, cache->head_dim, p.rt, grid, s);
    else
        launch_rows<BF16>(a, cache->head_dim, p.rt, grid, s);
    return check_launch("attention_q8", s);
}

}  // extern "C"
