// Attention of each sequence's new tokens over its paged cache (oom_attn_chunk_paged): attn_tile.hpp
// over pages, then the merge of the row tiles whose keys were split.
#include <cmath>

#include "attn_tile.hpp"

namespace oom {

// The merge of split rows: a wave a (row, KV head), in turn over all of them. The parts' maxima give
// their weights e^((m_p - M) scale); out = sum_p w_p O_p / sum_p w_p l_p, in part order. The
// first parts' O are on their way before the weights are known: a row takes two round trips
// of loads, its entry and then everything.
template <int D>
__global__ void __launch_bounds__(256) attn_rows_merge_kernel(TileArgs a, int64_t max_items) {
    constexpr int CPL = D / 64, EARLY = 8;  // columns a lane, parts loaded at once
    typedef float cols_t __attribute__((ext_vector_type(CPL)));
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int64_t all = (int64_t)a.plan[ATTN_PLAN_MERGES] * a.Hkv;
    const int4* rows = reinterpret_cast<const int4*>(a.plan + ATTN_PLAN_HEAD + max_items * ATTN_ITEM_WORDS);
    const float c = a.scale * 1.44269504088896340736f;
    for (int64_t i = wave; i < all; i += gridDim.x * 4) {
        const int h = (int)(i % a.Hkv);
        const int4 e = rows[i / a.Hkv];
        const int n = e.w & 0xffff, stride = e.w >> 16;
        const int64_t pr = (int64_t)h * a.part_rows + e.z;
        const float* acc = a.part_acc + pr * D + CPL * lane;
        cols_t v[EARLY], A = {};
#pragma unroll
        for (int j = 0; j < EARLY; j++)
            if (j < n) v[j] = *reinterpret_cast<const cols_t*>(acc + (int64_t)j * stride * D);  // uniform
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
            const int m = min(64, n - p0);
            for (int j0 = 0; j0 < m; j0 += EARLY) {
                if (p0 + j0 > 0)
#pragma unroll
                    for (int j = 0; j < EARLY; j++)
                        if (p0 + j0 + j < n)
                            v[j] = *reinterpret_cast<const cols_t*>(acc + (int64_t)(p0 + j0 + j) * stride * D);
#pragma unroll
                for (int j = 0; j < EARLY; j++) {
                    if (j0 + j >= m) break;
                    const float wj = __shfl(w, j0 + j);
#pragma unroll
                    for (int x = 0; x < CPL; x++) A[x] = fmaf(v[j][x], wj, A[x]);
                }
            }
        }
        const float inv = e.y >> 30 ? 0.0f : 1.0f / L;
        const int64_t at = (int64_t)e.x * a.out_stride + (int64_t)(h * a.G + (e.y & 0xffff)) * D + CPL * lane;
#pragma unroll
        for (int x = 0; x < CPL; x++) {
            if (a.out_dtype == OOM_BF16) store_out<OOM_BF16>(a.out, at + x, A[x] * inv);
            else store_out<OOM_F32>(a.out, at + x, A[x] * inv);
        }
    }
}

template <int D>
static int launch_chunk(const TileArgs& a, const AttnPlanDims& p, bool exact, hipStream_t st) {
    const dim3 grid((uint32_t)(p.items * a.Hkv));
    launch_tiles<D, true>(a, grid, exact, st);
    if (int rc = launched("oom_attn_chunk_paged")) return rc;
    const dim3 mgrid((uint32_t)std::min<int64_t>(2048, cdiv(p.merge_rows * a.Hkv, 4)));
    hipLaunchKernelGGL((attn_rows_merge_kernel<D>), mgrid, dim3(256), 0, st, a, p.items);
    return launched("oom_attn_chunk_paged");
}

}  // namespace oom

extern "C" size_t oom_attn_chunk_paged_workspace_size(int T, int B, int heads, int kv_heads, int d) {
    if (T < 0 || B < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || d < 1) return 0;
    return (size_t)oom::attn_plan_dims(T, B, heads, kv_heads).part_rows * kv_heads * (d + 2) * sizeof(float) + 256;
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
    OOM_REQUIRE(scale > 0.0f && std::isfinite(scale), "oom_attn_chunk_paged: scale must be positive and finite");
    OOM_REQUIRE(q_stride >= (int64_t)heads * d && out_stride >= (int64_t)heads * d && q_stride % 8 == 0 &&
                    out_stride % 8 == 0,
                "oom_attn_chunk_paged: strides must be multiples of 8 elements, at least a token's heads");
    if (T == 0 || B == 0) return OOM_OK;
    OOM_REQUIRE(q && k_pages && v_pages && page_table && plan && out, "oom_attn_chunk_paged: null buffer");
    OOM_REQUIRE(aligned(q, 16) && aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(out, 16) && aligned(plan, 16),
                "oom_attn_chunk_paged: q, k_pages, v_pages, out and plan must be 16-byte aligned");
    const AttnPlanDims p = attn_plan_dims(T, B, heads, kv_heads);
    OOM_REQUIRE(p.items * kv_heads < (1ll << 31), "oom_attn_chunk_paged: too many tiles of rows");
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
    a.G = heads / kv_heads;
    a.Hkv = kv_heads;
    a.scale = scale;
    a.part_rows = p.part_rows;
    a.part_acc = reinterpret_cast<float*>(ws);
    a.part_ml = a.part_acc + p.part_rows * kv_heads * d;
    const bool exact = q_dtype == OOM_F32 || out_dtype == OOM_F32;
    hipStream_t st = as_stream(stream);
    if (d == 64) return launch_chunk<64>(a, p, exact, st);
    if (d == 128) return launch_chunk<128>(a, p, exact, st);
    return launch_chunk<256>(a, p, exact, st);
}
