// Attention of tiles of query rows over 64-key tiles in LDS: the device core of
// oom_attn_prompt (packed prompts, K and V rows as the projections wrote them) and
// oom_attn_chunk_paged (new tokens over paged caches).
//
// A row is one (token, query head) pair: the G query heads that share a KV head are packed
// beside each other, row t G + g, so every row of a tile reads the same K and V and the
// rows of a tile span few tokens, whose causal bounds nearly agree.
//
//  * Scores S^T = K Q^T on v_mfma_f32_32x32x16_bf16 (keys on M): lane l ends with 16 keys of
//    row l % 32 a 32-key step, so the softmax of a row stays inside two lanes; its maximum
//    costs one half-wave swap a tile and its sum none before the end.
//  * O^T = V^T P^T on the same instruction (dims on M). The keys of a product may be summed
//    in any order that both operands share: P stays in the registers where the scores left
//    it, and V takes that order through transposing LDS reads (ds_read_b64_tr_b16, four keys
//    of one dim a lane).
//  * Running maximum m and sum l in fp32, base-2 exponentials: p = 2^(s c - m c), c = scale
//    log2 e, one fused multiply-add; for c > 1, where a finite score times c may be infinite, 2^((s -
//    m) c). O is rescaled only when some row's maximum grew by more than a factor of 2^8: until
//    then the older maximum keeps every p below 2^8, which fp32 sums hold as well.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace oom {

typedef __bf16 tbf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 tbf16x2 __attribute__((ext_vector_type(2)));
typedef float tf32x2 __attribute__((ext_vector_type(2)));
typedef float tf32x16 __attribute__((ext_vector_type(16)));
typedef short ts16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ts16x4* tr_ptr_t;
typedef __attribute__((address_space(3))) void* t_lds_t;

constexpr float T_GROW = 8.0f;  // growth of a row's maximum (log2) that rescales O

// What one block works on: an entry of the plan (attn_plan.hip).
struct AttnItem {
    int q0;    // first token row of the sequence
    int row0;  // first packed row of the tile within the sequence
    int rows;  // its rows
    int off;   // position of the sequence's first new token
    int k0, k1;  // its keys [k0, k1), k0 a multiple of 64
    int part;  // first row of its partial, -1: the only split, writes out
    int seq;
};
static_assert(sizeof(AttnItem) == 4 * ATTN_ITEM_WORDS, "plan item");

struct TileArgs {
    const void* q;
    int64_t q_stride;  // elements between tokens
    int q_dtype, out_dtype;
    void* out;
    int64_t out_stride;
    const uint16_t* k;  // prompt: rows [T, Hkv, d]; paged: the pages
    const uint16_t* v;
    int64_t k_stride, v_stride;  // prompt: elements between tokens
    const int32_t* table;        // paged: [B, max_pages]
    int max_pages, n_pages, page_size;
    const int32_t* plan;
    int plan_sign;
    int G, Hkv;
    float scale;
    float* part_ml;   // [Hkv][part rows][2]: maximum score and sum
    float* part_acc;  // [Hkv][part rows][d]
    int64_t part_rows;
};

// Rows that a bad page index, or a key past the item's end, reads: zeros.
static __device__ __align__(16) uint16_t t_zero_row[256];

__device__ __forceinline__ uint32_t t_pack(float a, float b) {
    const tf32x2 f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, tbf16x2));  // RNE
}

__device__ __forceinline__ void t_barrier() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// A K or V tile in LDS: 64 rows (keys) of d bf16, in 16-byte chunks, C = d / 8 a row, each row's
// chunks permuted by an exclusive or with a value of the row, so that the lanes of a read,
// which take the same chunks of consecutive rows, meet different banks. A direct-to-LDS load
// writes lane l's 16 bytes at its base + 16 l, so the permutation is in the global addresses.
//   K: chunk ^ (row % 16 (8 for d = 64)): 16 consecutive rows' same chunk in 16 places
//   V: the transposing read takes 4 rows x 2 chunks a 16-lane group
template <int D>
struct TileLay {
    static constexpr int C = D / 8, ROWB = D * 2, BYTES = 64 * ROWB;
    static constexpr int RPI = 64 / C;  // rows an instruction loads
    static __device__ __forceinline__ int kx(int row) { return row & (C < 16 ? C - 1 : 15); }
    static __device__ __forceinline__ int vx(int row) { return D == 64 ? ((row >> 1) & 1) * 2 : (row & 3) * 4; }
};

// 16 bytes a lane straight into LDS: lane l's land at lds + 16 l (lds uniform). In assembly, so that
// the compiler does not wait for these loads before LDS reads of another stage: the kernel's own
// waits and barriers order them. The address is a uniform base plus a 32-bit offset a lane.
__device__ __forceinline__ void t_load_lds(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base)
                 : "memory", "m0");
}
__device__ __forceinline__ void t_load_lds(const void* at, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(at)
                 : "memory", "m0");
}
// This wave's loads into LDS, and its LDS reads and writes, are done. A builtin, which the compiler's
// own accounting sees: past it, no load of its own is outstanding, and it places no wait for one
// inside the tile loop, where it would wait for the loads into LDS too.
__device__ __forceinline__ void t_wait_loads() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// This wave's LDS reads and writes are done; its loads into LDS may be on their way.
__device__ __forceinline__ void t_wait_lds() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0); vmcnt and expcnt left at their maxima
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Where a run of keys lies in its page: byte offset from the head's first row of page 0, or -1 (a bad
// page, or past the item's keys).
__device__ __forceinline__ int64_t page_offset(const TileArgs& a, const int32_t* table, int key, int k1, int row_bytes) {
    if (key >= k1) return -1;
    const uint32_t pi = (uint32_t)key / (uint32_t)a.page_size;
    const int page = table[pi];
    if (page < 0 || page >= a.n_pages) return -1;
    return ((int64_t)page * a.Hkv * a.page_size + (key - (int)pi * a.page_size)) * row_bytes;
}
__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// Loads of one 64-key tile: wave w of NW takes 64 / NW rows of K and of V, which lie in one page.
// Over pages, lane i holds the place of the wave's rows of tile i (modulo 64): looked up a tile at a
// time, each tile waited for its page index before its loads could go out (512 tokens over 16 Ki
// keys 312 us, so 284).
template <int D, int NW, bool PAGED>
struct TileSrc {
    typedef TileLay<D> L;
    static constexpr int WR = 64 / NW, NI = WR / L::RPI;  // rows and instructions a wave
    static_assert(NI >= 1 && WR <= 16 && 16 % WR == 0, "whole instructions, one 16-key run");
    const uint8_t *k, *v;
    int64_t ks, vs;  // bytes between rows
    const int32_t* table;
    int first, k1;  // the wave's first key; the item's end
    int64_t places;
    uint32_t ko[NI], vo[NI];  // byte offsets of this lane from the wave's first row

    __device__ __forceinline__ void init(const TileArgs& a, const AttnItem& it, int h, int lane, int wave) {
        k1 = it.k1;
        first = it.k0 + WR * wave;
        k = reinterpret_cast<const uint8_t*>(a.k);
        v = reinterpret_cast<const uint8_t*>(a.v);
        if constexpr (PAGED) {
            ks = vs = L::ROWB;
            table = a.table + (size_t)it.seq * a.max_pages;
            k += (int64_t)h * a.page_size * L::ROWB;
            v += (int64_t)h * a.page_size * L::ROWB;
        } else {
            ks = 2 * a.k_stride;
            vs = 2 * a.v_stride;
            k += (int64_t)it.q0 * ks + h * L::ROWB;
            v += (int64_t)it.q0 * vs + h * L::ROWB;
        }
#pragma unroll
        for (int n = 0; n < NI; n++) {
            const int r = n * L::RPI + lane / L::C, c = lane % L::C;
            ko[n] = (uint32_t)(r * ks) + 16 * (c ^ L::kx(WR * wave + r));
            vo[n] = (uint32_t)(r * vs) + 16 * (c ^ L::vx(WR * wave + r));
        }
    }

    // The wave's rows of tile t into its places kt and vt (LDS byte addresses of its first row in the
    // K and the V tile).
    __device__ __forceinline__ void load(const TileArgs& a, int t, int lane, uint32_t kt, uint32_t vt) {
        const int key = first + 64 * t;
        int64_t kat, vat;
        bool ok = key < k1;
        if constexpr (PAGED) {
            if (t % 64 == 0) {
                places = page_offset(a, table, key + 64 * lane, k1, L::ROWB);
                __builtin_amdgcn_s_waitcnt(0);
            }
            kat = vat = lane_value(places, t % 64);
            ok = kat >= 0;
        } else {
            kat = key * ks;
            vat = key * vs;
        }
        const uint8_t *kb = k + kat, *vb = v + vat;
        if (ok && key + WR <= k1) {  // uniform
#pragma unroll
            for (int n = 0; n < NI; n++) t_load_lds(kb, ko[n], kt + n * 1024);
#pragma unroll
            for (int n = 0; n < NI; n++) t_load_lds(vb, vo[n], vt + n * 1024);
            return;
        }
        const uint8_t* z = (const uint8_t*)t_zero_row + 16 * (lane % L::C);
#pragma unroll
        for (int n = 0; n < NI; n++) {
            const bool in = ok && key + n * L::RPI + lane / L::C < k1;
            t_load_lds(in ? kb + ko[n] : z, kt + n * 1024);
            t_load_lds(in ? vb + vo[n] : z, vt + n * 1024);
        }
    }
};

// bf16 pairs whose exponent is all ones (infinity or NaN) in either half: nonzero.
__device__ __forceinline__ uint32_t t_nonfinite(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
// The pair with such halves cleared.
__device__ __forceinline__ uint32_t t_finite(uint32_t w) {
    const uint32_t b = t_nonfinite(w);
    uint32_t m = (b >> 15) * 0xffffu;  // 0x00010001 flags to half masks
    return w & ~m;
}

__device__ __forceinline__ tbf16x8 t_finite8(tbf16x8 v) {
    const uint4 w = __builtin_bit_cast(uint4, v);
    return __builtin_bit_cast(tbf16x8, make_uint4(t_finite(w.x), t_finite(w.y), t_finite(w.z), t_finite(w.w)));
}

typedef float tf32x4 __attribute__((ext_vector_type(4)));

// The matrix instruction of M rows: S^T tiles of M keys x M rows over 512 / M dims, O^T tiles of M
// dims x M rows over 512 / M keys. Lane l holds row l % M, and of a result's keys or dims the
// four 4 (l / M) .. + 3 of each run of 256 / M: element i of a result is its key (dim)
// (256 / M) (i / 4) + 4 (l / M) + i % 4.
template <int M>
struct Mx;
template <>
struct Mx<32> {
    typedef tf32x16 acc;
    static __device__ __forceinline__ acc mul(tbf16x8 a, tbf16x8 b, acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mx<16> {
    typedef tf32x4 acc;
    static __device__ __forceinline__ acc mul(tbf16x8 a, tbf16x8 b, acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// TERMS 1: bf16 queries and outputs: the products take Q as it is and P rounded to bf16 (its
// relative error, at most 2^-8 a key and averaged over the keys, is of the size of the
// output's own rounding; the sum l is that of the rounded p). TERMS 3: fp32 on either side: Q
// and P enter as three exact bf16 terms each (hi + mid + lo), so products are exact and only
// fp32 sums round.
// A wave scores KEYS keys of a tile and holds DO of the output's dims: all of both, but for pair_block().
template <int D, int TERMS, int M, int KEYS = ATTN_KEYS, int DO = D>
struct RowState {
    static constexpr int KD = 512 / M;    // dims (keys) a product sums over
    static constexpr int E = M * M / 64;  // elements of a result a lane
    static constexpr int NS = KEYS / M;   // results a tile of scores
    static constexpr int NO = DO / M;     // results of the output
    typedef typename Mx<M>::acc acc;
    tbf16x8 q[TERMS][D / KD];
    acc o[NO];
    acc sc[NS];  // scores of the present tile
    float m, l;
    int pos;    // the last key this lane's row sees
    bool live;  // the lane has a row
};
// The key of element i of score result n, without the lane's 4 (l / M).
template <int M>
constexpr int score_key(int n, int i) { return M * n + (256 / M) * (i / 4) + i % 4; }

template <int D, int TERMS, int M, int KEYS, int DO>
__device__ __forceinline__ void rows_init(RowState<D, TERMS, M, KEYS, DO>& s, const TileArgs& a, const AttnItem& it, int h, int wrow,
                                          int lane) {
    const int r = wrow + lane % M, part = lane / M;
    s.live = r < it.rows;
    const uint32_t row = (uint32_t)(it.row0 + (s.live ? r : 0)), tok = row / (uint32_t)a.G, g = row - tok * a.G;
    s.pos = it.off + (int)tok;
    s.m = -INFINITY;
    s.l = 0.0f;
#pragma unroll
    for (int d = 0; d < DO / M; d++) s.o[d] = typename Mx<M>::acc{};
    constexpr int KD = 512 / M;
    const int64_t at = (int64_t)(it.q0 + (int)tok) * a.q_stride + (int64_t)(h * a.G + (int)g) * D + 8 * part;
    if constexpr (TERMS == 1) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(a.q) + at;
#pragma unroll
        for (int c = 0; c < D / KD; c++)
            s.q[0][c] = __builtin_bit_cast(tbf16x8, *reinterpret_cast<const uint4*>(p + KD * c));
    } else {
        const bool wide = a.q_dtype == OOM_F32;  // uniform
        const uint8_t* p = reinterpret_cast<const uint8_t*>(a.q) + at * (wide ? 4 : 2);
        uint4 raw[D / KD][2];
#pragma unroll
        for (int c = 0; c < D / KD; c++) {
            raw[c][0] = *reinterpret_cast<const uint4*>(p + KD * c * (wide ? 4 : 2));
            raw[c][1] = wide ? *reinterpret_cast<const uint4*>(p + KD * c * 4 + 16) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < D / KD; c++) {
            const uint4 x = raw[c][0], y = raw[c][1];
            const uint32_t n[8] = {x.x << 16, x.x & 0xffff0000u, x.y << 16, x.y & 0xffff0000u,
                                   x.z << 16, x.z & 0xffff0000u, x.w << 16, x.w & 0xffff0000u};
            const uint32_t f4[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = __uint_as_float(wide ? f4[e] : n[e]);
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    w[e] = t_pack(f[2 * e], f[2 * e + 1]);
                    f[2 * e] -= __uint_as_float(w[e] << 16);  // exact: the remainder of a round to nearest
                    f[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
                }
                s.q[t][c] = __builtin_bit_cast(tbf16x8, make_uint4(w[0], w[1], w[2], w[3]));
            }
        }
    }
}

// Scores of one K tile from LDS. MASKED: some key of the tile is hidden from some row, by a later position
// or past the item's keys (last: the last one that the lane's row sees). BAD_K, with three terms: K
// holds infinities or NaN, which meet the first term alone; the others may be zero or of the
// other sign. V holds none (the kernel takes them out).
template <bool MASKED, bool BAD_K, int D, int TERMS, int M, int KEYS, int DO>
__device__ __forceinline__ void tile_scores(RowState<D, TERMS, M, KEYS, DO>& s, const uint8_t* kt, int last, int lane) {
    typedef TileLay<D> L;
    typedef RowState<D, TERMS, M, KEYS, DO> S;
    const int part = lane / M;
    const uint8_t* krow = kt + (lane % M) * L::ROWB;
    const int kx = L::kx(lane % M);  // rows M apart have the same
#pragma unroll
    for (int st = 0; st < D / S::KD; st++) {
        const int chunk = (S::KD / 8 * st + part) ^ kx;
        tbf16x8 ka[S::NS], kf[S::NS];
#pragma unroll
        for (int n = 0; n < S::NS; n++) {
            const uint4 kv = *reinterpret_cast<const uint4*>(krow + M * n * L::ROWB + 16 * chunk);
            ka[n] = __builtin_bit_cast(tbf16x8, kv);
            if constexpr (TERMS > 1) kf[n] = BAD_K ? t_finite8(ka[n]) : ka[n];
            if (st == 0) s.sc[n] = typename S::acc{};
        }
        // products of one sum apart from each other: the next would wait for the last one's result
#pragma unroll
        for (int t = TERMS - 1; t >= 0; t--)
#pragma unroll
            for (int n = 0; n < S::NS; n++) s.sc[n] = Mx<M>::mul(t > 0 ? kf[n] : ka[n], s.q[t][st], s.sc[n]);
    }
    if constexpr (MASKED) {
#pragma unroll
        for (int n = 0; n < S::NS; n++)
#pragma unroll
            for (int i = 0; i < S::E; i++)
                if (score_key<M>(n, i) + 4 * part > last) s.sc[n][i] = -INFINITY;
    }
}

// The largest of v over the lanes of a row.
template <int M>
__device__ __forceinline__ float row_max(float v) {
    if constexpr (M == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int M>
__device__ __forceinline__ float row_sum(float v) {
    if constexpr (M == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The running maximum; O and l rescaled where it grew enough. Returns what the tile's exponents
// subtract.
template <int D, int TERMS, int M, int KEYS>
__device__ __forceinline__ float tile_maximum(RowState<D, TERMS, M, KEYS>& s, float c) {
    typedef RowState<D, TERMS, M, KEYS> S;
    float mx = s.sc[0][0];
#pragma unroll
    for (int n = 0; n < S::NS; n++)
#pragma unroll
        for (int i = 0; i < S::E; i++) mx = fmaxf(mx, s.sc[n][i]);
    mx = row_max<M>(mx);
    if (__any((mx - s.m) * c > T_GROW || s.m == -INFINITY)) {
        const float mn = fmaxf(s.m, mx);
        const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((s.m - mn) * c);
        s.m = mn;
        s.l *= f;
#pragma unroll
        for (int d = 0; d < D / M; d++)
#pragma unroll
            for (int i = 0; i < S::E; i++) s.o[d][i] *= f;
    }
    float m0 = s.m == -INFINITY ? 0.0f : s.m;
    if (c > 1.0f) {  // uniform
#pragma unroll
        for (int n = 0; n < S::NS; n++)
#pragma unroll
            for (int i = 0; i < S::E; i++) s.sc[n][i] -= m0;
        m0 = 0.0f;
    }
    return m0 * c;
}

// The tile's weights p = 2^(s c - mb), their sum, and O += V^T P^T.
template <int D, int TERMS, int M, int KEYS>
__device__ __forceinline__ void tile_values(RowState<D, TERMS, M, KEYS>& s, const uint8_t* vt, float c, float mb, int lane) {
    typedef TileLay<D> L;
    typedef RowState<D, TERMS, M, KEYS> S;
    const tbf16x2 ones = __builtin_bit_cast(tbf16x2, 0x3f803f80u);
    const int part = lane / M, r4 = (lane & 15) >> 2;
    const uint8_t* vrow = vt + (4 * part + r4) * L::ROWB + 8 * (lane & 1);
    const int vc = (M == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((lane & 3) >> 1), vx = L::vx(4 * part + r4);
#pragma unroll
    for (int w = 0; w < KEYS / S::KD; w++) {
        // the lane's 8 keys of this product: two runs of four, 256 / M apart
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int e = 8 * w + j;  // of the lane's E NS scores, in order
            p[j] = __builtin_amdgcn_exp2f(fmaf(s.sc[e / S::E][e % S::E], c, -mb));
        }
        if constexpr (TERMS > 1) {
#pragma unroll
            for (int j = 0; j < 8; j++) s.l += p[j];
        }
        tbf16x8 pb[TERMS];
#pragma unroll
        for (int t = 0; t < TERMS; t++) {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                b[j] = t_pack(p[2 * j], p[2 * j + 1]);
                if (TERMS == 1) s.l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(tbf16x2, b[j]), ones, s.l, false);
                if (t + 1 < TERMS) {
                    p[2 * j] -= __uint_as_float(b[j] << 16);  // exact: the remainder of a round to nearest
                    p[2 * j + 1] -= __uint_as_float(b[j] & 0xffff0000u);
                }
            }
            pb[t] = __builtin_bit_cast(tbf16x8, make_uint4(b[0], b[1], b[2], b[3]));
        }
        constexpr int DB = TERMS == 1 ? 1 : D / M < 4 ? D / M : 4;  // results whose products alternate
#pragma unroll
        for (int d0 = 0; d0 < D / M; d0 += DB) {
            tbf16x8 vv[DB];
#pragma unroll
            for (int i = 0; i < DB; i++) {
                const uint8_t* va = vrow + S::KD * w * L::ROWB + 16 * ((M / 8 * (d0 + i) + vc) ^ vx);
                const ts16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)va);
                const ts16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)(va + 256 / M * L::ROWB));
                const uint2 w0 = __builtin_bit_cast(uint2, v0), w1 = __builtin_bit_cast(uint2, v1);
                vv[i] = __builtin_bit_cast(tbf16x8, make_uint4(w0.x, w0.y, w1.x, w1.y));
            }
#pragma unroll
            for (int t = TERMS - 1; t >= 0; t--)
#pragma unroll
                for (int i = 0; i < DB; i++) s.o[d0 + i] = Mx<M>::mul(vv[i], pb[t], s.o[d0 + i]);
        }
    }
    if constexpr (TERMS > 1) {
        // V's operands of the next results are read before the present ones' products
        constexpr int MFMA = 0x008, LDSR = 0x100, DB = D / M < 4 ? D / M : 4;
        __builtin_amdgcn_sched_group_barrier(LDSR, 2 * DB, 0);
#pragma unroll
        for (int i = 0; i < KEYS / S::KD * (D / M) / DB; i++) {
            __builtin_amdgcn_sched_group_barrier(LDSR, 2 * DB, 0);
            __builtin_amdgcn_sched_group_barrier(MFMA, TERMS * DB, 0);
        }
    }
}

// The infinities and NaN of a V tile to the rows that see their key: a hidden key has no part in a
// row, whatever its value holds, and its weight of zero times an infinity would be NaN.
template <int D, int TERMS, int M, int KEYS, int DO>
__device__ __forceinline__ void tile_bad_values(RowState<D, TERMS, M, KEYS, DO>& s, const uint8_t* vt, int last, int lane,
                                                int keys = KEYS, int dim0 = 0) {
    typedef TileLay<D> L;
    const int part = lane / M;
    for (int key = 0; key < keys; key++) {
        if (!__any(key <= last)) break;
#pragma unroll
        for (int d = 0; d < DO / M; d++)
#pragma unroll
            for (int e = 0; e < M * M / 256; e++) {
                const int dim = dim0 + M * d + (256 / M) * e + 4 * part;
                const uint2 w = *reinterpret_cast<const uint2*>(vt + key * L::ROWB + 16 * ((dim / 8) ^ L::vx(key)) +
                                                                2 * (dim & 7));
                const uint32_t b0 = w.x & ~t_finite(w.x), b1 = w.y & ~t_finite(w.y);
                if (key <= last) {
                    s.o[d][4 * e] += __uint_as_float(b0 << 16);
                    s.o[d][4 * e + 1] += __uint_as_float(b0 & 0xffff0000u);
                    s.o[d][4 * e + 2] += __uint_as_float(b1 << 16);
                    s.o[d][4 * e + 3] += __uint_as_float(b1 & 0xffff0000u);
                }
            }
    }
}

// The token row and the head of the group of packed row r of the sequence.
__device__ __forceinline__ int64_t row_at(const TileArgs& a, const AttnItem& it, int h, int D, int r) {
    const uint32_t row = (uint32_t)(it.row0 + r), tok = row / (uint32_t)a.G, g = row - tok * a.G;
    return (int64_t)(it.q0 + (int)tok) * a.out_stride + (int64_t)(h * a.G + (int)g) * D;
}

// out = O / l of the wave's rows, or their partial (O, m, l) for the merge. A row that sees no key
// gives zeros. Lanes hold columns of rows: they go through LDS (the wave's share of the tiles' places,
// which no wave reads any more) so that a store covers whole rows, 1 KB at a time; chunks of 16
// bytes are permuted within a row against bank conflicts. (Stored from the registers, 8 or 16
// bytes a row and instruction: 2 % slower on short prompts.)
template <int D, int TERMS, int M, int KEYS, int DO>
__device__ __forceinline__ void rows_store(RowState<D, TERMS, M, KEYS, DO>& s, const TileArgs& a, const AttnItem& it, int h,
                                           int wrow, int lane, uint8_t* lds, int dim0 = 0) {
    const int r = lane % M, part = lane / M;
    s.l = row_sum<M>(s.l);
    const bool wide = it.part >= 0 || a.out_dtype == OOM_F32;  // uniform
    const int64_t pr = (int64_t)h * a.part_rows + it.part + wrow;
    if (it.part >= 0 && dim0 == 0 && part == 0 && s.live) *reinterpret_cast<float2*>(a.part_ml + 2 * (pr + r)) = make_float2(s.m, s.l);
    const float f = it.part >= 0 ? 1.0f : s.pos < 0 ? 0.0f : 1.0f / s.l;
#pragma unroll
    for (int d = 0; d < DO / M; d++)
#pragma unroll
        for (int e = 0; e < M * M / 256; e++) {
            const float x0 = s.o[d][4 * e] * f, x1 = s.o[d][4 * e + 1] * f, x2 = s.o[d][4 * e + 2] * f,
                        x3 = s.o[d][4 * e + 3] * f;
            const int dim = M * d + 256 / M * e + 4 * part;
            if (wide)
                *reinterpret_cast<float4*>(lds + r * DO * 4 + 16 * ((dim / 4) ^ (r & 15))) = make_float4(x0, x1, x2, x3);
            else
                *reinterpret_cast<uint2*>(lds + r * DO * 2 + 16 * ((dim / 8) ^ (r & (DO / 8 - 1) & 15)) + 2 * (dim & 7)) =
                    make_uint2(t_pack(x0, x1), t_pack(x2, x3));
        }
    wave_lds_order();
    if (wide) {
        constexpr int C = DO / 4;  // chunks a row
#pragma unroll
        for (int i = 0; i < M * C / 64; i++) {
            const int row = (64 * i + lane) / C, ch = (64 * i + lane) % C;
            if (wrow + row >= it.rows) continue;
            const float4 v = *reinterpret_cast<const float4*>(lds + row * DO * 4 + 16 * (ch ^ (row & 15)));
            float* to = it.part >= 0 ? a.part_acc + (pr + row) * D
                                     : reinterpret_cast<float*>(a.out) + row_at(a, it, h, D, wrow + row);
            *reinterpret_cast<float4*>(to + dim0 + 4 * ch) = v;
        }
    } else {
        constexpr int C = DO / 8;
#pragma unroll
        for (int i = 0; i < M * C / 64; i++) {
            const int row = (64 * i + lane) / C, ch = (64 * i + lane) % C;
            if (wrow + row >= it.rows) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(lds + row * DO * 2 + 16 * (ch ^ (row & (C - 1) & 15)));
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + row_at(a, it, h, D, wrow + row) + dim0 + 8 * ch) =
                v;
        }
    }
}

// NW waves of M rows a block: a whole tile of 128 rows, or part of one; block i takes part i / Hkv
// for KV head i % Hkv (consecutive blocks run on different XCDs, so with 8 KV heads each L2 holds
// one head's K and V).
// K and V tiles go through LDS in two stages, one barrier a tile: past it, every wave has done
// with the stage that the next tile's loads now fill, and those have a whole tile to arrive.
// Two blocks a CU (d up to 128) or two waves a SIMD take turns on the matrix cores and the
// vector units. bad_lds: per stage, K and V hold infinities or NaN.
template <int D>
constexpr int tile_lds() { return 4 * TileLay<D>::BYTES; }  // stage 0: K, V; stage 1: K, V

template <int D, int TERMS, int M, int NW, bool PAGED>
__device__ __forceinline__ void tile_block(const TileArgs& a, uint32_t index, uint8_t* tiles, uint32_t (&bad_lds)[4]) {
    typedef TileLay<D> L;
    constexpr int ROWS = NW * M, PARTS = ATTN_ROWS / ROWS;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int)(index % (uint32_t)a.Hkv), block = (int)(index / (uint32_t)a.Hkv);
    const int item = block / PARTS, row_b = block % PARTS * ROWS;  // the block's first row of the tile
    AttnItem it = reinterpret_cast<const AttnItem*>(a.plan + ATTN_PLAN_HEAD)[item];
    if (a.plan[ATTN_PLAN_SIGN] != a.plan_sign || item >= a.plan[ATTN_PLAN_ITEMS] || row_b >= it.rows) return;
    const int wrow = row_b + M * wave;
    const bool has = wrow < it.rows;  // uniform
    const float c = a.scale * 1.44269504088896340736f;
    // Half tiles are twice the blocks that the plan split the keys for: a block takes two splits of its
    // tile (an even one and the next), so that they still run at once, and leaves the second's
    // partial empty (200 fp32 tokens over 2500 keys beside 15 single ones: 56.8 us, so 53.7).
    int empty = 0;  // rows from its partial to the second's, if there is one
    if constexpr (PARTS > 1 && PAGED) {
        const int split = a.plan[ATTN_PLAN_SPLIT], keys = it.off + 1 + (int)((uint32_t)(it.row0 + it.rows - 1) / (uint32_t)a.G);
        if (it.part >= 0 && it.k0 / split % 2 != 0) return;
        if (it.part >= 0 && it.k1 < keys) {
            it.k1 = min(keys, it.k1 + split);
            empty = it.rows;
        }
    }
    // no row of the block sees keys past its last row's position
    if constexpr (PARTS > 1)
        it.k1 = min(it.k1, it.off + 1 + (int)((uint32_t)(it.row0 + min(row_b + ROWS, it.rows) - 1) / (uint32_t)a.G));
    TileSrc<D, NW, PAGED> src;
    src.init(a, it, h, lane, wave);
    if (threadIdx.x < 4) bad_lds[threadIdx.x] = 0;
    const uint32_t mine = (uint32_t)(uintptr_t)(t_lds_t)tiles + wave * (L::BYTES / NW);  // LDS address of the wave's rows
    if (it.k0 < it.k1) src.load(a, 0, lane, mine, mine + L::BYTES);
    RowState<D, TERMS, M> s;
    rows_init(s, a, it, h, wrow, lane);
    __syncthreads();  // bad_lds is cleared
    // the wave's last position; the tiles that every row of the block sees whole come first
    const int pos_hi = it.off + (int)((uint32_t)(it.row0 + min(wrow + M - 1, it.rows - 1)) / (uint32_t)a.G);
    const int block_lo = it.off + (int)((uint32_t)(it.row0 + row_b) / (uint32_t)a.G);
    const int whole = it.k0 + (max(0, min(it.k1, block_lo + 1) - it.k0) & ~63);
    int key0 = it.k0;
    uint32_t stage = 0;

    // K's (three terms) and V's infinities and NaN in the wave's part of the tile
    const auto look = [&]() {
        uint32_t bk = 0, bv = 0;
#pragma unroll
        for (int n = 0; n < L::BYTES / NW / 1024; n++) {
            const uint8_t* at = tiles + stage + wave * (L::BYTES / NW) + n * 1024 + 16 * lane;
            const uint4 w = *reinterpret_cast<const uint4*>(at + L::BYTES);
            bv |= t_nonfinite(w.x) | t_nonfinite(w.y) | t_nonfinite(w.z) | t_nonfinite(w.w);
            if constexpr (TERMS > 1) {
                const uint4 y = *reinterpret_cast<const uint4*>(at);
                bk |= t_nonfinite(y.x) | t_nonfinite(y.y) | t_nonfinite(y.z) | t_nonfinite(y.w);
            }
        }
        uint32_t* const bad = bad_lds + (stage ? 2 : 0);
        if (bk) bad[0] = 1;
        if (bv) bad[1] = 1;
        t_wait_lds();
    };
    const auto step = [&](auto masked_tile) {
        constexpr bool MASKED = decltype(masked_tile)::value;
        const uint8_t* const kt = tiles + stage;
        uint8_t* const vt = tiles + stage + L::BYTES;
        t_wait_loads();
        if constexpr (MASKED || TERMS > 1) look();
        t_barrier();
        if (key0 + 64 < it.k1) {
            const uint32_t to = mine + (stage ^ (2 * L::BYTES));
            src.load(a, (key0 + 64 - it.k0) / 64, lane, to, to + L::BYTES);
        }
        const bool sees = has && (!MASKED || key0 <= pos_hi);  // uniform
        const int last = MASKED ? min(s.pos, it.k1 - 1) - key0 : 63;
        if (sees) {
            if (TERMS > 1 && bad_lds[stage ? 2 : 0] != 0) tile_scores<MASKED, true>(s, kt, last, lane);
            else tile_scores<MASKED, false>(s, kt, last, lane);
        }
        const float mb = sees ? tile_maximum(s, c) : 0.0f;
        if ((MASKED || TERMS > 1) && bad_lds[stage ? 3 : 1] != 0) {  // uniform over the block; rare
            if (sees) tile_bad_values(s, vt, last, lane);
            __syncthreads();
#pragma unroll
            for (int n = 0; n < L::BYTES / NW / 1024; n++) {
                uint4* p = reinterpret_cast<uint4*>(vt + wave * (L::BYTES / NW) + n * 1024 + 16 * lane);
                *p = __builtin_bit_cast(uint4, t_finite8(__builtin_bit_cast(tbf16x8, *p)));
            }
            if (threadIdx.x == 0) bad_lds[stage ? 3 : 1] = 0;
            __syncthreads();
        }
        if (sees) tile_values(s, vt, c, mb, lane);
    };
    for (; key0 < whole; key0 += 64, stage ^= 2 * L::BYTES) step(std::false_type{});
    for (; key0 < it.k1; key0 += 64, stage ^= 2 * L::BYTES) step(std::true_type{});
    __syncthreads();  // every wave is done with the tiles
    static_assert(4 * L::BYTES >= NW * M * D * 4, "the rows fit the tiles' places");
    if (has) rows_store(s, a, it, h, wrow, lane, tiles + wave * (M * D * 4));
    if (empty > 0 && lane < M && s.live)
        *reinterpret_cast<float2*>(a.part_ml + 2 * ((int64_t)h * a.part_rows + it.part + empty + wrow + lane)) =
            make_float2(-INFINITY, 0.0f);
}

// d 256 in one term, whose 16-row waves above would each read the whole tile from LDS for half the
// products: a pair of waves (w, w + 4) has 32 rows. Each scores half of the tile's keys, and their
// weights meet in LDS; then each sums all keys' values into half of the dims. So a wave reads
// half of K and half of V, and its Q and half of O leave room for two waves a SIMD. The pair
// keeps the same maxima: the weights are taken with those of the tiles before, and only where a
// row of the block outgrew its (by T_GROW; a row's first keys do) do the pairs exchange maxima
// and take the weights again.
// (2048 and 40 tokens at 24/2 heads: 74 us with 16-row waves, 67 so. A tile takes 1.7 us a CU, and 1.2
// with its products left out: the issue of its loads, barriers, LDS round trips and softmax.)
struct PairLds {
    uint4 p[8][2][64];  // a wave's weights: the operands of its two products a tile
    float mx[8][32];    // its rows' maxima, where some row's grew
    uint32_t grew[2];   // some row's did, by the tile's parity
    uint32_t bad[2];    // V holds infinities or NaN, by stage
};

// The N products before this are issued with their operands' LDS reads (R each) up to 6 products ahead.
template <int N, int R>
__device__ __forceinline__ void reads_ahead() {
    constexpr int MFMA = 0x008, LDSR = 0x100, AHEAD = 6;
    __builtin_amdgcn_sched_group_barrier(LDSR, R * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; i++) {
        __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
        __builtin_amdgcn_sched_group_barrier(LDSR, R, 0);
    }
    __builtin_amdgcn_sched_group_barrier(MFMA, AHEAD, 0);
}

template <bool PAGED>
__device__ __forceinline__ void pair_block(const TileArgs& a, uint32_t index, uint8_t* tiles, PairLds& x) {
    constexpr int D = 256, M = 32, NW = 8, DO = D / 2;
    typedef TileLay<D> L;
    typedef RowState<D, 1, M, 32, DO> S;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int)(index % (uint32_t)a.Hkv), item = (int)(index / (uint32_t)a.Hkv);
    const AttnItem it = reinterpret_cast<const AttnItem*>(a.plan + ATTN_PLAN_HEAD)[item];
    if (a.plan[ATTN_PLAN_SIGN] != a.plan_sign || item >= a.plan[ATTN_PLAN_ITEMS]) return;
    const int part = wave / 4, wrow = M * (wave % 4);  // the wave's half of the keys, then of the dims
    const bool has = wrow < it.rows;                   // uniform
    const float c = a.scale * 1.44269504088896340736f;
    TileSrc<D, NW, PAGED> src;
    src.init(a, it, h, lane, wave);
    if (threadIdx.x < 2) x.grew[threadIdx.x] = x.bad[threadIdx.x] = 0;
    const uint32_t mine = (uint32_t)(uintptr_t)(t_lds_t)tiles + wave * (L::BYTES / NW);
    if (it.k0 < it.k1) src.load(a, 0, lane, mine, mine + L::BYTES);
    S s;
    rows_init(s, a, it, h, wrow, lane);
    __syncthreads();  // the flags are cleared
    const int pos_hi = it.off + (int)((uint32_t)(it.row0 + min(wrow + M - 1, it.rows - 1)) / (uint32_t)a.G);
    const int block_lo = it.off + (int)((uint32_t)it.row0 / (uint32_t)a.G);
    const int whole = it.k0 + (max(0, min(it.k1, block_lo + 1) - it.k0) & ~63);
    int key0 = it.k0;
    uint32_t odd = 0;  // the tile's parity: its stage
    // where a lane's first K chunk and V rows are in a tile of stage 0: chunks differ in bits 4 to 8 of the
    // place, which the permutations combine by exclusive or, and the tiles are 32 KB each
    const uint32_t k_at = (32 * part + lane % M) * L::ROWB + 16 * ((lane / M) ^ L::kx(lane % M));
    const int vr = 4 * (lane / M) + ((lane & 15) >> 2);
    const uint32_t v_at = L::BYTES + (32 * part + vr) * L::ROWB + 8 * (lane & 1) +
                          16 * ((DO / 8 * part + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ L::vx(vr));
    tbf16x8 pb[2];
    // p = 2^(s c - m c) of the wave's scores, for itself and for its partner
    const auto weights = [&]() {
        const float m0 = s.m == -INFINITY ? 0.0f : s.m, sub = c > 1.0f ? m0 : 0.0f, mb = c > 1.0f ? 0.0f : m0 * c;
#pragma unroll
        for (int w = 0; w < 2; w++) {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float s0 = s.sc[0][8 * w + 2 * j], s1 = s.sc[0][8 * w + 2 * j + 1];
                b[j] = t_pack(__builtin_amdgcn_exp2f(fmaf(s0 - sub, c, -mb)), __builtin_amdgcn_exp2f(fmaf(s1 - sub, c, -mb)));
            }
            const uint4 v = make_uint4(b[0], b[1], b[2], b[3]);
            pb[w] = __builtin_bit_cast(tbf16x8, v);
            x.p[wave][w][lane] = v;
        }
    };
    const auto step = [&](auto masked_tile) {
        constexpr bool MASKED = decltype(masked_tile)::value;
        uint8_t* const vt = tiles + odd * (2 * L::BYTES) + L::BYTES;
        t_wait_loads();
        if constexpr (MASKED) {  // V's infinities and NaN in the wave's part of the tile
            uint32_t bv = 0;
#pragma unroll
            for (int n = 0; n < L::BYTES / NW / 1024; n++) {
                const uint4 w = *reinterpret_cast<const uint4*>(vt + wave * (L::BYTES / NW) + n * 1024 + 16 * lane);
                bv |= t_nonfinite(w.x) | t_nonfinite(w.y) | t_nonfinite(w.z) | t_nonfinite(w.w);
            }
            if (bv) x.bad[odd] = 1;
            t_wait_lds();
        }
        t_barrier();
        if (key0 + 64 < it.k1) {
            const uint32_t to = mine + (odd ^ 1) * (2 * L::BYTES);
            src.load(a, (key0 + 64 - it.k0) / 64, lane, to, to + L::BYTES);
        }
        const bool sees = has && (!MASKED || key0 <= pos_hi);  // uniform, and the same for the pair
        const int last = MASKED ? min(s.pos, it.k1 - 1) - key0 : 63;
        float mx = -INFINITY;
        if (sees) {
            s.sc[0] = typename S::acc{};
#pragma unroll
            for (int st = 0; st < D / S::KD; st++) {
                const tbf16x8 k8 = *reinterpret_cast<const tbf16x8*>(tiles + (k_at ^ (odd * (2 * L::BYTES)) ^ 32 * st));
                s.sc[0] = Mx<M>::mul(k8, s.q[0][st], s.sc[0]);
            }
            reads_ahead<D / S::KD, 1>();
            if constexpr (MASKED) {
#pragma unroll
                for (int i = 0; i < S::E; i++)
                    if (score_key<M>(part, i) + 4 * (lane / M) > last) s.sc[0][i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < S::E; i++) mx = fmaxf(mx, s.sc[0][i]);
            mx = row_max<M>(mx);
            if (__any((mx - s.m) * c > T_GROW)) x.grew[odd] = 1;
            weights();
        }
        if (threadIdx.x == 0) x.grew[odd ^ 1] = 0;  // read before this tile's first barrier, set past the next's
        t_wait_lds();
        t_barrier();
        if (x.grew[odd]) {  // uniform over the block; rare
            if (sees && lane < M) x.mx[wave][lane] = mx;
            t_wait_lds();
            t_barrier();
            if (sees) {
                const float mn = fmaxf(s.m, fmaxf(mx, x.mx[wave ^ 4][lane % M]));
                const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((s.m - mn) * c);
                s.m = mn;
                s.l *= f;
#pragma unroll
                for (int d = 0; d < S::NO; d++)
#pragma unroll
                    for (int i = 0; i < S::E; i++) s.o[d][i] *= f;
                weights();
            }
            t_wait_lds();
            t_barrier();
        }
        if (MASKED && x.bad[odd]) {  // uniform over the block; rare
            if (sees) tile_bad_values(s, vt, last, lane, ATTN_KEYS, DO * part);
            __syncthreads();
#pragma unroll
            for (int n = 0; n < L::BYTES / NW / 1024; n++) {
                uint4* p = reinterpret_cast<uint4*>(vt + wave * (L::BYTES / NW) + n * 1024 + 16 * lane);
                *p = __builtin_bit_cast(uint4, t_finite8(__builtin_bit_cast(tbf16x8, *p)));
            }
            if (threadIdx.x == 0) x.bad[odd] = 0;
            __syncthreads();
        }
        if (sees) {
            const tbf16x2 ones = __builtin_bit_cast(tbf16x2, 0x3f803f80u);
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const uint4 v = __builtin_bit_cast(uint4, pb[w]);
                for (const uint32_t b : {v.x, v.y, v.z, v.w})
                    s.l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(tbf16x2, b), ones, s.l, false);
            }
            // 16 keys a product: those of the wave's own half, then its partner's
            tbf16x8 p2[2];
#pragma unroll
            for (int w = 0; w < 2; w++) p2[w] = __builtin_bit_cast(tbf16x8, x.p[wave ^ 4][w][lane]);
#pragma unroll
            for (int w = 0; w < 4; w++)
#pragma unroll
                for (int d = 0; d < S::NO; d++) {
                    const uint8_t* va = tiles + ((v_at ^ (odd * (2 * L::BYTES)) ^ 64 * d) ^ (w < 2 ? 0 : 32 * L::ROWB)) +
                                        16 * (w % 2) * L::ROWB;
                    const uint2 w0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)va));
                    const uint2 w1 =
                        __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)(va + 8 * L::ROWB)));
                    s.o[d] = Mx<M>::mul(__builtin_bit_cast(tbf16x8, make_uint4(w0.x, w0.y, w1.x, w1.y)),
                                        w < 2 ? pb[w] : p2[w - 2], s.o[d]);
                }
            reads_ahead<4 * S::NO, 2>();
        }
    };
    for (; key0 < whole; key0 += 64, odd ^= 1) step(std::false_type{});
    for (; key0 < it.k1; key0 += 64, odd ^= 1) step(std::true_type{});
    __syncthreads();  // every wave is done with the tiles and the weights
    float* const sums = reinterpret_cast<float*>(x.p);
    sums[64 * wave + lane] = s.l;
    __syncthreads();
    s.l += sums[64 * (wave ^ 4) + lane];
    static_assert(4 * L::BYTES >= NW * M * DO * 4, "the rows fit the tiles' places");
    if (has) rows_store(s, a, it, h, wrow, lane, tiles + wave * (M * DO * 4), DO * part);
}

// Rows a wave: 32 in one term (d 256: pair_block()), 16 for three terms, whose Q of 32 rows leaves no
// registers for a second wave on the SIMD. Waves a block: a tile's rows, but half of them for
// three terms up to d 128, so that two blocks fit a CU and do not wait at the same barriers (LDS
// holds one block at d 256).
template <int D, int TERMS>
struct TileShape {
    static constexpr bool PAIRS = D == 256 && TERMS == 1;
    static constexpr int M = TERMS == 1 ? 32 : 16;
    static constexpr int NW = D <= 128 ? 4 : 8;  // 64 NW threads: tile_threads()
    static constexpr int PARTS = PAIRS ? 1 : ATTN_ROWS / (M * NW);  // blocks a tile
};

template <int D>
constexpr int tile_threads() { return D <= 128 ? 256 : 512; }

template <int D, int TERMS, bool PAGED>
__global__ void __launch_bounds__(tile_threads<D>(), 2) attn_tile_kernel(TileArgs a) {
    typedef TileShape<D, TERMS> S;
    __shared__ __align__(16) uint8_t tiles[tile_lds<D>()];
    if constexpr (S::PAIRS) {
        __shared__ PairLds pairs;
        pair_block<PAGED>(a, blockIdx.x, tiles, pairs);
    } else {
        __shared__ uint32_t bad_lds[4];
        tile_block<D, TERMS, S::M, S::NW, PAGED>(a, blockIdx.x, tiles, bad_lds);
    }
}

template <int D, int TERMS, bool PAGED>
void launch_tiles(const TileArgs& a, int64_t items, hipStream_t st) {
    typedef TileShape<D, TERMS> S;
    hipLaunchKernelGGL((attn_tile_kernel<D, TERMS, PAGED>), dim3((uint32_t)(items * a.Hkv * S::PARTS)), dim3(64 * S::NW), 0,
                       st, a);
}

}  // namespace oom
