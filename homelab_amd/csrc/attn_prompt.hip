// Causal attention of packed prompts (oom_attn_prompt): attn_tile.hpp over the K and V rows of the
// prompts' own tokens.
#include "attn_tile.hpp"

namespace oom {

template <int D>
static int launch_prompt(const TileArgs& a, int64_t items, bool exact, hipStream_t st) {
    if (exact) launch_tiles<D, 3, false>(a, items, st);
    else launch_tiles<D, 1, false>(a, items, st);
    return launched("oom_attn_prompt");
}

}  // namespace oom

extern "C" int oom_attn_prompt(const void* q, int q_dtype, int64_t q_stride, const uint16_t* k, int64_t k_stride,
                               const uint16_t* v, int64_t v_stride, const int32_t* plan, int T, int B, int heads,
                               int kv_heads, int d, float scale, void* out, int out_dtype, int64_t out_stride,
                               void* stream) {
    using namespace oom;
    OOM_REQUIRE(d == 64 || d == 128 || d == 256, "oom_attn_prompt: head_dim must be 64, 128 or 256");
    OOM_REQUIRE(kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && heads <= 4096,
                "oom_attn_prompt: heads must be a multiple of kv_heads, at most 4096");
    OOM_REQUIRE(T >= 0 && B >= 0 && B <= ATTN_MAXB && (int64_t)T * heads < (1ll << 31),
                "oom_attn_prompt: at most 4096 sequences, and fewer than 2^31 rows of heads");
    OOM_REQUIRE(q_dtype == OOM_F32 || q_dtype == OOM_BF16, "oom_attn_prompt: q_dtype");
    OOM_REQUIRE(out_dtype == OOM_F32 || out_dtype == OOM_BF16, "oom_attn_prompt: out_dtype");
    OOM_REQUIRE(scale >= 0x1p-60f && scale <= 0x1p60f, "oom_attn_prompt: scale must be from 2^-60 to 2^60");
    OOM_REQUIRE(q_stride >= (int64_t)heads * d && out_stride >= (int64_t)heads * d &&
                    k_stride >= (int64_t)kv_heads * d && v_stride >= (int64_t)kv_heads * d,
                "oom_attn_prompt: strides smaller than a token's heads");
    OOM_REQUIRE(q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 && out_stride % 8 == 0 &&
                    k_stride < (1ll << 25) && v_stride < (1ll << 25),
                "oom_attn_prompt: strides must be multiples of 8 elements, K's and V's under 2^25");
    if (T == 0 || B == 0) return OOM_OK;
    OOM_REQUIRE(q && k && v && plan && out, "oom_attn_prompt: null buffer");
    OOM_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && aligned(plan, 16),
                "oom_attn_prompt: q, k, v, out and plan must be 16-byte aligned");
    const AttnPlanDims p = attn_plan_dims(T, B, heads, kv_heads, d);
    OOM_REQUIRE(p.tiles * kv_heads < (1ll << 30), "oom_attn_prompt: too many tiles of rows");
    TileArgs a = {};
    a.q = q;
    a.q_stride = q_stride;
    a.q_dtype = q_dtype;
    a.out_dtype = out_dtype;
    a.out = out;
    a.out_stride = out_stride;
    a.k = k;
    a.v = v;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.plan = plan;
    a.plan_sign = attn_plan_sign(T, B, heads, kv_heads, d, 0, 0);
    a.G = heads / kv_heads;
    a.Hkv = kv_heads;
    a.scale = scale;
    const bool exact = q_dtype == OOM_F32 || out_dtype == OOM_F32;
    hipStream_t st = as_stream(stream);
    if (d == 64) return launch_prompt<64>(a, p.tiles, exact, st);
    if (d == 128) return launch_prompt<128>(a, p.tiles, exact, st);
    return launch_prompt<256>(a, p.tiles, exact, st);
}
