// Attention of each sequence's new tokens over its paged cache (oom_attn_chunk_paged): attn_tile.hpp
// over pages, then the merge of the row tiles whose keys were split.
#include "attn_few.hpp"

namespace oom {

// The merge of split rows: a wave a (row, KV head), in turn over all of them. The parts' maxima give
// their weights e^((m_p - M) scale); out = sum_p w_p O_p / sum_p w_p l_p. A load takes the row of
// 256 / d parts, 16 bytes a lane; the first 8 loads' parts are on their way before the weights
// are known, so a row takes two round trips, its entry and then everything.
template <int D>
__global__ void __launch_bounds__(256) attn_rows_merge_kernel(TileArgs a, const int4* rows) {
    constexpr int LPP = D / 4, PP = 64 / LPP, EARLY = 8;  // lanes a part, parts a load, loads at once
    const int lane = threadIdx.x & 63, sub = lane / LPP, col = lane % LPP * 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int64_t all = a.plan[ATTN_PLAN_SIGN] == a.plan_sign ? (int64_t)a.plan[ATTN_PLAN_MERGES] * a.Hkv : 0;
    const float c = a.scale * 1.44269504088896340736f;
    for (int64_t i = wave; i < all; i += gridDim.x * 4) {
        const int h = (int)(i % a.Hkv);
        const int4 e = rows[i / a.Hkv];
        const int n = e.w & 0xffff, stride = e.w >> 16;
        const int64_t pr = (int64_t)h * a.part_rows + e.z;
        const float* acc = a.part_acc + pr * D + col;
        float4 v[EARLY];
        float A[4] = {};
        const auto load = [&](int p0) {
#pragma unroll
            for (int j = 0; j < EARLY; j++)
                if (p0 + PP * j < n)  // uniform
                    v[j] = *reinterpret_cast<const float4*>(acc + (int64_t)min(p0 + PP * j + sub, n - 1) * stride * D);
        };
        load(0);
        float M = -INFINITY, L = 0.0f;
        for (int p0 = 0; p0 < n; p0 += 64)
            if (p0 + lane < n) M = fmaxf(M, a.part_ml[2 * (pr + (int64_t)(p0 + lane) * stride)]);
        M = wave_max(M);
        for (int p0 = 0; p0 < n; p0 += 64) {
            float w = 0.0f, l = 0.0f;
            if (p0 + lane < n) {
                const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (pr + (int64_t)(p0 + lane) * stride));
                w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ml.x - M) * c);
                l = ml.y * w;
            }
            L += wave_sum(l);
            for (int q0 = 0; q0 < min(64, n - p0); q0 += PP * EARLY) {
                if (p0 + q0 > 0) load(p0 + q0);
#pragma unroll
                for (int j = 0; j < EARLY; j++) {
                    const int p = q0 + PP * j + sub;
                    const float wj = __shfl(w, p & 63);
                    if (p < 64 && p0 + p < n && wj != 0.0f) {  // (an empty partial's O is not written)
                        A[0] = fmaf(v[j].x, wj, A[0]);
                        A[1] = fmaf(v[j].y, wj, A[1]);
                        A[2] = fmaf(v[j].z, wj, A[2]);
                        A[3] = fmaf(v[j].w, wj, A[3]);
                    }
                }
            }
        }
#pragma unroll
        for (int o = 32; o >= LPP; o >>= 1)
#pragma unroll
            for (int x = 0; x < 4; x++) A[x] += lane_xor_n(A[x], o, lane);
        if (sub > 0) continue;
        const float inv = e.y >> 30 ? 0.0f : 1.0f / L;
        const int64_t at = (int64_t)e.x * a.out_stride + (int64_t)(h * a.G + (e.y & 0xffff)) * D + col;
        if (a.out_dtype == OOM_BF16)
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + at) =
                make_uint2(t_pack(A[0] * inv, A[1] * inv), t_pack(A[2] * inv, A[3] * inv));
        else
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at) =
                make_float4(A[0] * inv, A[1] * inv, A[2] * inv, A[3] * inv);
    }
}

// The kernels that a batch may need. Tiles: where max_q new tokens have more rows than a few-row
// sequence, or the batch's lone sequence is none by its kind.
template <int D, int TERMS>
static void launch_rows(const TileArgs& a, const AttnPlanDims& p, int64_t T, int B, int max_q, hipStream_t st) {
    const bool few = attn_has_few(T, B, a.G, D), tiles = !few || (int64_t)max_q * a.G > attn_few_rows(D);
    if constexpr (D <= 128)
        if (tiles && few) return launch_mixed<D, TERMS>(a, p, st);
    if (tiles) launch_tiles<D, TERMS, true>(a, p.items, st);
    if (few) launch_few<D, TERMS>(a, p, st);
}

template <int D>
static int launch_chunk(const TileArgs& a, const AttnPlanDims& p, int T, int B, int max_q, bool exact, hipStream_t st) {
    if (exact) launch_rows<D, 3>(a, p, T, B, max_q, st);
    else launch_rows<D, 1>(a, p, T, B, max_q, st);
    if (int rc = launched("oom_attn_chunk_paged")) return rc;
    const int4* rows = reinterpret_cast<const int4*>(a.plan + ATTN_PLAN_HEAD + (p.items + p.few_items) * ATTN_ITEM_WORDS);
    const dim3 grid((uint32_t)std::min<int64_t>(2048, cdiv(p.merge_rows * a.Hkv, 4)));
    hipLaunchKernelGGL((attn_rows_merge_kernel<D>), grid, dim3(256), 0, st, a, rows);
    return launched("oom_attn_chunk_paged");
}

}  // namespace oom

extern "C" size_t oom_attn_chunk_paged_workspace_size(int T, int B, int heads, int kv_heads, int d) {
    if (T < 0 || B < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || d < 1) return 0;
    return (size_t)oom::attn_plan_dims(T, B, heads, kv_heads, d).part_rows * kv_heads * (d + 2) * sizeof(float) + 256;
}

extern "C" int oom_attn_chunk_paged(const void* q, int q_dtype, int64_t q_stride, const uint16_t* k_pages,
                                    const uint16_t* v_pages, const int32_t* page_table, int max_pages, int n_pages,
                                    int page_size, const int32_t* plan, int T, int B, int max_q, int heads, int kv_heads,
                                    int d, float scale, void* out, int out_dtype, int64_t out_stride, void* ws,
                                    size_t ws_bytes, void* stream) {
    using namespace oom;
    OOM_REQUIRE(d == 64 || d == 128 || d == 256, "oom_attn_chunk_paged: head_dim must be 64, 128 or 256");
    OOM_REQUIRE(kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && heads <= 4096,
                "oom_attn_chunk_paged: heads must be a multiple of kv_heads, at most 4096");
    OOM_REQUIRE(T >= 0 && B >= 0 && B <= ATTN_MAXB && (int64_t)T * heads < (1ll << 31),
                "oom_attn_chunk_paged: at most 4096 sequences, and fewer than 2^31 rows of heads");
    OOM_REQUIRE(max_q >= 1 || T == 0, "oom_attn_chunk_paged: max_q must be >= 1");
    OOM_REQUIRE(page_size >= 16 && page_size % 16 == 0, "oom_attn_chunk_paged: page_size must be a multiple of 16");
    OOM_REQUIRE(n_pages >= 1 && max_pages >= 1 && (int64_t)max_pages * page_size <= ATTN_MAX_KEYS,
                "oom_attn_chunk_paged: n_pages and max_pages must be >= 1, a sequence at most 128 Mi keys");
    OOM_REQUIRE(q_dtype == OOM_F32 || q_dtype == OOM_BF16, "oom_attn_chunk_paged: q_dtype");
    OOM_REQUIRE(out_dtype == OOM_F32 || out_dtype == OOM_BF16, "oom_attn_chunk_paged: out_dtype");
    OOM_REQUIRE(scale >= 0x1p-60f && scale <= 0x1p60f, "oom_attn_chunk_paged: scale must be from 2^-60 to 2^60");
    OOM_REQUIRE(q_stride >= (int64_t)heads * d && out_stride >= (int64_t)heads * d && q_stride % 8 == 0 &&
                    out_stride % 8 == 0,
                "oom_attn_chunk_paged: strides must be multiples of 8 elements, at least a token's heads");
    if (T == 0 || B == 0) return OOM_OK;
    OOM_REQUIRE(q && k_pages && v_pages && page_table && plan && out, "oom_attn_chunk_paged: null buffer");
    OOM_REQUIRE(aligned(q, 16) && aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(out, 16) && aligned(plan, 16),
                "oom_attn_chunk_paged: q, k_pages, v_pages, out and plan must be 16-byte aligned");
    const AttnPlanDims p = attn_plan_dims(T, B, heads, kv_heads, d);
    OOM_REQUIRE((p.items + p.few_items) * kv_heads < (1ll << 30), "oom_attn_chunk_paged: too many tiles of rows");
    if (!ws || ws_bytes < oom_attn_chunk_paged_workspace_size(T, B, heads, kv_heads, d))
        return fail(OOM_ERR_WORKSPACE,
                    "oom_attn_chunk_paged: workspace smaller than oom_attn_chunk_paged_workspace_size()");
    OOM_REQUIRE(aligned(ws, 256), "oom_attn_chunk_paged: workspace must be 256-byte aligned");
    TileArgs a = {};
    a.q = q;
    a.q_stride = q_stride;
    a.q_dtype = q_dtype;
    a.out_dtype = out_dtype;
    a.out = out;
    a.out_stride = out_stride;
    a.k = k_pages;
    a.v = v_pages;
    a.table = page_table;
    a.max_pages = max_pages;
    a.n_pages = n_pages;
    a.page_size = page_size;
    a.plan = plan;
    a.plan_sign = attn_plan_sign(T, B, heads, kv_heads, d, max_pages, page_size);
    a.G = heads / kv_heads;
    a.Hkv = kv_heads;
    a.scale = scale;
    a.part_rows = p.part_rows;
    a.part_acc = reinterpret_cast<float*>(ws);
    a.part_ml = a.part_acc + p.part_rows * kv_heads * d;
    const bool exact = q_dtype == OOM_F32 || out_dtype == OOM_F32;
    hipStream_t st = as_stream(stream);
    if (d == 64) return launch_chunk<64>(a, p, T, B, max_q, exact, st);
    if (d == 128) return launch_chunk<128>(a, p, T, B, max_q, exact, st);
    return launch_chunk<256>(a, p, T, B, max_q, exact, st);
}
