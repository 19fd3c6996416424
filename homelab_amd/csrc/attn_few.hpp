// Attention of sequences with few new rows (at most attn_few_rows(): a decode step, a few drafted
// tokens) over their paged caches: bound by the stream of K and V, not by products.
//
// Where attn_tile.hpp gives each wave of a block other rows of the same keys, here every wave has
// the same rows (16 or 32) and other keys: wave w of NW takes the 32-key tiles w, w + NW, ... of
// its block's item, from LDS places of its own, so no barrier stands in the loop and every wave
// streams. A wave has one place each for K and V, filled again as soon as its products have
// read it: the next tile's K arrives beside the present one's values, and two blocks a CU (8
// waves of 16 KB at d 128) keep more than enough bytes under way. At the end the waves' (maximum,
// sum, O) meet in LDS.
#pragma once

#include "attn_tile.hpp"

namespace oom {

constexpr int FK = 32;  // keys a tile

template <int D>
constexpr int few_waves() { return D == 256 ? 2 : 4; }

// s_waitcnt vmcnt(N): this wave's loads but the newest N are done.
template <int N>
__device__ __forceinline__ void f_wait_loads() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

template <int D, int TERMS, int M>
__device__ __forceinline__ void few_rows(const TileArgs& a, const AttnItem& it, int h, uint8_t* lds,
                                         float (&mlds)[few_waves<D>()][32], float (&llds)[few_waves<D>()][32]) {
    typedef TileLay<D> L;
    constexpr int NW = few_waves<D>();
    constexpr int TB = FK * L::ROWB;    // bytes of a K or V tile
    constexpr int NI = 16 / L::RPI;     // loads of 16 rows
    constexpr int PIECES = FK / 16;     // runs of 16 keys, each in one page
    constexpr int LOADS = PIECES * NI;  // of a K or V tile
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float c = a.scale * 1.44269504088896340736f;
    const int32_t* const table = a.table + (size_t)it.seq * a.max_pages;
    const uint8_t* const kb = (const uint8_t*)a.k + (int64_t)h * a.page_size * D * 2;
    const uint8_t* const vb = (const uint8_t*)a.v + (int64_t)h * a.page_size * D * 2;
    const uint8_t* const kt = lds + wave * 2 * TB;
    uint8_t* const vt = lds + wave * 2 * TB + TB;
    const uint32_t k_at = (uint32_t)(uintptr_t)(t_lds_t)lds + wave * 2 * TB, v_at = k_at + TB;
    // tile t of the wave starts at key0(t); its run x's place is in lane 2 t + x (t modulo 32)
    const auto key0 = [&](int t) { return it.k0 + FK * (wave + NW * t); };
    const int left = it.k1 - key0(0);
    const int n = left > 0 ? (left + FK * NW - 1) / (FK * NW) : 0;  // the wave's tiles
    int64_t found = -1;
    const auto find_places = [&](int t0) {
        found = page_offset(a, table, key0(t0 + lane / PIECES) + 16 * (lane % PIECES), it.k1, L::ROWB);
    };
    uint32_t ko[NI], vo[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int r = i * L::RPI + lane / L::C, ch = lane % L::C;
        ko[i] = r * L::ROWB + 16 * (ch ^ L::kx(r));
        vo[i] = r * L::ROWB + 16 * (ch ^ L::vx(r));
    }
    // K's or V's rows of tile t (base: kb or vb; off: ko or vo) into LDS at `to`
    const auto load = [&](int t, const uint8_t* base, const uint32_t (&off)[NI], uint32_t to) {
#pragma unroll
        for (int x = 0; x < PIECES; x++) {
            const int key = key0(t) + 16 * x;
            const int64_t place = lane_value(found, (PIECES * t + x) & 63);
            const bool ok = place >= 0;
            const uint8_t* at = base + place;
            if (ok && key + 16 <= it.k1) {  // uniform
#pragma unroll
                for (int i = 0; i < NI; i++) t_load_lds(at, off[i], to + x * 16 * L::ROWB + i * 1024);
            } else {
                const uint8_t* z = (const uint8_t*)t_zero_row + 16 * (lane % L::C);
#pragma unroll
                for (int i = 0; i < NI; i++)
                    t_load_lds(ok && key + i * L::RPI + lane / L::C < it.k1 ? at + off[i] : z,
                               to + x * 16 * L::ROWB + i * 1024);
            }
        }
    };
    if (n > 0) find_places(0);
    RowState<D, TERMS, M, FK> s;
    rows_init(s, a, it, h, 0, lane);
    t_wait_loads();  // the compiler's own loads are done: from here on the count is the tiles'
    if (n > 0) {
        load(0, kb, ko, k_at);
        load(0, vb, vo, v_at);
    }
    const int lo = it.off + (int)((uint32_t)it.row0 / (uint32_t)a.G);  // the first row's position
    const auto look = [&](const uint8_t* tile) {
        uint32_t b = 0;
#pragma unroll
        for (int i = 0; i < TB / 1024; i++) {
            const uint4 w = *reinterpret_cast<const uint4*>(tile + i * 1024 + 16 * lane);
            b |= t_nonfinite(w.x) | t_nonfinite(w.y) | t_nonfinite(w.z) | t_nonfinite(w.w);
        }
        return __any(b != 0);
    };
    const auto step = [&](int t, auto masked_tile) {
        constexpr bool MASKED = decltype(masked_tile)::value;
        const bool more = t + 1 < n;
        const int last = MASKED ? min(s.pos, it.k1 - 1) - key0(t) : FK - 1;
        f_wait_loads<LOADS>();  // K; V's loads are the newer ones
        if (TERMS > 1 && look(kt)) tile_scores<MASKED, true>(s, kt, last, lane);
        else tile_scores<MASKED, false>(s, kt, last, lane);
        if (more && (t + 1) % (64 / PIECES) == 0) {
            find_places(t + 1);
            t_wait_loads();
        }
        if (more) {
            t_wait_lds();
            load(t + 1, kb, ko, k_at);
        }
        const float mb = tile_maximum(s, c);
        if (more) f_wait_loads<LOADS>();
        else f_wait_loads<0>();
        if ((MASKED || TERMS > 1) && look(vt)) {  // rare
            tile_bad_values(s, vt, last, lane);
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < TB / 1024; i++) {
                uint4* p = reinterpret_cast<uint4*>(vt + i * 1024 + 16 * lane);
                *p = __builtin_bit_cast(uint4, t_finite8(__builtin_bit_cast(tbf16x8, *p)));
            }
            wave_lds_order();
        }
        tile_values(s, vt, c, mb, lane);
        if (more) {
            t_wait_lds();
            load(t + 1, vb, vo, v_at);
        }
    };
    for (int t = 0; t < n; t++) {
        if (key0(t) + FK - 1 > lo || key0(t) + FK > it.k1) step(t, std::true_type{});
        else step(t, std::false_type{});
    }
    // ---- the waves' results meet ----
    s.l = row_sum<M>(s.l);
    __syncthreads();
    float* const olds = reinterpret_cast<float*>(lds);  // [NW][M][D]
    static_assert(2 * TB >= M * D * 4, "a wave's O fits its places");
    const int row = lane % M, part = lane / M;
    if (part == 0) {
        mlds[wave][row] = s.m;
        llds[wave][row] = s.l;
    }
#pragma unroll
    for (int d = 0; d < D / M; d++)
#pragma unroll
        for (int e = 0; e < M * M / 256; e++)
            *reinterpret_cast<float4*>(olds + (wave * M + row) * D + M * d + 256 / M * e + 4 * part) =
                make_float4(s.o[d][4 * e], s.o[d][4 * e + 1], s.o[d][4 * e + 2], s.o[d][4 * e + 3]);
    __syncthreads();
    // four columns a thread
    for (int i = threadIdx.x; i < it.rows * (D / 4); i += 64 * NW) {
        const int r = i / (D / 4), col = i % (D / 4) * 4;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; w++) mx = fmaxf(mx, mlds[w][r]);
        float sum = 0.0f;
        float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float m = mlds[w][r], f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mx) * c);
            const float4 v = *reinterpret_cast<const float4*>(olds + (w * M + r) * D + col);
            sum = fmaf(llds[w][r], f, sum);
            o.x = fmaf(v.x, f, o.x);
            o.y = fmaf(v.y, f, o.y);
            o.z = fmaf(v.z, f, o.z);
            o.w = fmaf(v.w, f, o.w);
        }
        const uint32_t rr = (uint32_t)(it.row0 + r), tok = rr / (uint32_t)a.G, g = rr - tok * a.G;
        if (it.part >= 0) {
            const int64_t pr = (int64_t)h * a.part_rows + it.part + r;
            if (col == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * pr) = make_float2(mx, sum);
            *reinterpret_cast<float4*>(a.part_acc + pr * D + col) = o;
            continue;
        }
        const float inv = it.off + (int)tok < 0 ? 0.0f : 1.0f / sum;
        const int64_t at = (int64_t)(it.q0 + (int)tok) * a.out_stride + (int64_t)(h * a.G + (int)g) * D + col;
        if (a.out_dtype == OOM_BF16)
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + at) =
                make_uint2(t_pack(o.x * inv, o.y * inv), t_pack(o.z * inv, o.w * inv));
        else
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at) =
                make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
}

template <int D>
constexpr int few_lds() { return few_waves<D>() * 2 * FK * TileLay<D>::ROWB; }

// Block i takes few-row item i / Hkv for KV head i % Hkv, with as many rows a wave as it needs.
template <int D, int TERMS>
__device__ __forceinline__ void few_block(const TileArgs& a, uint32_t index, int64_t max_items, uint8_t* lds,
                                          float (&mlds)[few_waves<D>()][32], float (&llds)[few_waves<D>()][32]) {
    const int h = (int)(index % (uint32_t)a.Hkv), item = (int)(index / (uint32_t)a.Hkv);
    const AttnItem it = reinterpret_cast<const AttnItem*>(a.plan + ATTN_PLAN_HEAD + max_items * ATTN_ITEM_WORDS)[item];
    if (a.plan[ATTN_PLAN_SIGN] != a.plan_sign || item >= a.plan[ATTN_PLAN_FEW]) return;
    if constexpr (attn_few_rows(D) > 16)
        if (it.rows > 16) return few_rows<D, TERMS, 32>(a, it, h, lds, mlds, llds);
    few_rows<D, TERMS, 16>(a, it, h, lds, mlds, llds);
}

template <int D, int TERMS>
__global__ void __launch_bounds__(64 * few_waves<D>(), D == 128 && TERMS == 3 ? 1 : 2)
    attn_few_kernel(TileArgs a, int64_t max_items) {
    __shared__ __align__(16) uint8_t lds[few_lds<D>()];
    __shared__ float mlds[few_waves<D>()][32], llds[few_waves<D>()][32];
    few_block<D, TERMS>(a, blockIdx.x, max_items, lds, mlds, llds);
}

template <int D, int TERMS>
void launch_few(const TileArgs& a, const AttnPlanDims& p, hipStream_t st) {
    hipLaunchKernelGGL((attn_few_kernel<D, TERMS>), dim3((uint32_t)(p.few_items * a.Hkv)), dim3(64 * few_waves<D>()), 0, st, a,
                       p.items);
}

// Both kinds of a mixed batch in one launch (d up to 128: the same block and LDS): the tiles first,
// which are the longer, then the few-row sequences, which fill the CUs that the last tiles leave
// idle.
template <int D, int TERMS>
__global__ void __launch_bounds__(256, 2) attn_mixed_kernel(TileArgs a, int64_t max_items, uint32_t tile_blocks) {
    typedef TileShape<D, TERMS> S;
    static_assert(S::NW == 4 && few_waves<D>() == 4, "one block size");
    __shared__ __align__(16) uint8_t lds[tile_lds<D>() > few_lds<D>() ? tile_lds<D>() : few_lds<D>()];
    __shared__ float mlds[4][32], llds[4][32];
    __shared__ uint32_t bad_lds[4];
    if (blockIdx.x < tile_blocks) tile_block<D, TERMS, S::M, 4, true>(a, blockIdx.x, lds, bad_lds);
    else few_block<D, TERMS>(a, blockIdx.x - tile_blocks, max_items, lds, mlds, llds);
}

template <int D, int TERMS>
void launch_mixed(const TileArgs& a, const AttnPlanDims& p, hipStream_t st) {
    const uint32_t tiles = (uint32_t)(p.items * a.Hkv * TileShape<D, TERMS>::PARTS);
    hipLaunchKernelGGL((attn_mixed_kernel<D, TERMS>), dim3(tiles + (uint32_t)(p.few_items * a.Hkv)), dim3(256), 0, st, a, p.items,
                       tiles);
}

}  // namespace oom
