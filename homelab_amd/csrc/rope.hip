// Rotary positions: oom_rope on rows of heads, and oom_rope_append_paged, which rotates a step's
// queries and keys and writes the keys and values into the paged cache.
//
// The pair (u, w) of dims i of a head turns by theta = pos f_i: (u cos - w sin, u sin + w cos).
// An angle of a far position needs more bits than fp32 has: at position 10^6 its error would be
// 0.06 rad. So a frequency is held as a 64-bit fraction of a full turn, f_i / 2 pi * 2^64, and
// theta in turns is pos times it modulo 2^64: one integer product, exact but for the
// fraction's own rounding (pos * 2^-54 turns at worst). sin and cos of the turn, as a
// signed fraction, then round like any fp32 function's. The products are fp32, rounded
// once to the output's type.
#include <cmath>

#include "common.hpp"

namespace oom {

struct RopeArgs {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;  // elements between tokens
    const int32_t* positions;
    const int64_t* slots;
    const uint64_t* turns;
    int rot, d, T, H, Hkv;
    float magnitude, sign;
    void* out;
    int64_t out_stride;
    uint16_t *kp, *vp;
    int64_t n_slots;
    int page_size;
};

__device__ __forceinline__ void turn_sincos(int pos, uint64_t f, float& s, float& c) {
    const int64_t t = (int64_t)((uint64_t)(int64_t)pos * f);  // turns * 2^64, in [-1/2, 1/2)
    const float half_turns = (float)(int32_t)(t >> 32) * 0x1p-31f;  // angle / pi in [-1, 1), 2^-32 turns off at most
    sincospif(half_turns, &s, &c);
}

// One thread a pair (or two elements past rot) of the queries, then of the keys, then of the
// values. Reading both before writing either, it may work in place.
template <int XDT, int ODT, bool APPEND>
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs a, int layout) {
    const int t = blockIdx.y, heads = a.H + (APPEND ? 2 * a.Hkv : 0), half = a.rot / 2;
    const int e = blockIdx.x * 256 + threadIdx.x;
    if (e >= heads * (a.d / 2)) return;
    const int hd = e / (a.d / 2), u = e - hd * (a.d / 2);
    const void* x = a.q;
    int64_t at = t * a.q_stride + (int64_t)hd * a.d;
    if (APPEND && hd >= a.H + a.Hkv) {
        x = a.v;
        at = t * a.v_stride + (int64_t)(hd - a.H - a.Hkv) * a.d;
    } else if (APPEND && hd >= a.H) {
        x = a.k;
        at = t * a.k_stride + (int64_t)(hd - a.H) * a.d;
    }
    int i = 2 * u, j = 2 * u + 1;
    if (layout == OOM_ROPE_HALF && u < half) {
        i = u;
        j = u + half;
    }
    float y = load_act<XDT>(x, at + i), z = load_act<XDT>(x, at + j);
    if (u < half && hd < a.H + a.Hkv) {
        float s, c;
        turn_sincos(a.positions[t], a.turns[u], s, c);
        s *= a.sign * a.magnitude;
        c *= a.magnitude;
        const float y0 = y;
        y = fmaf(y0, c, -(z * s));
        z = fmaf(y0, s, z * c);
    }
    if (!APPEND || hd < a.H) {
        const int64_t to = t * a.out_stride + (int64_t)hd * a.d;
        store_out<ODT>(a.out, to + i, y);
        store_out<ODT>(a.out, to + j, z);
        return;
    }
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.n_slots) return;
    const int g = hd < a.H + a.Hkv ? hd - a.H : hd - a.H - a.Hkv;
    uint16_t* p = (hd < a.H + a.Hkv ? a.kp : a.vp) +
                  ((slot / a.page_size * a.Hkv + g) * a.page_size + slot % a.page_size) * a.d;
    p[i] = f32_to_bf16(y);
    p[j] = f32_to_bf16(z);
}

}  // namespace oom

extern "C" int oom_rope_table(const OomRope* rope, uint64_t* turns, size_t n, float* magnitude) {
    using namespace oom;
    OOM_REQUIRE(rope && turns && magnitude, "oom_rope_table: null buffer");
    const int rot = (int)rope->rot_dim;
    OOM_REQUIRE(rope->rot_dim >= 2 && rope->rot_dim <= 1024 && rot % 2 == 0, "oom_rope_table: rot_dim must be even, 2 to 1024");
    OOM_REQUIRE(rope->base > 1.0 && std::isfinite(rope->base), "oom_rope_table: base must be above 1");
    OOM_REQUIRE(rope->scaling == OOM_ROPE_PLAIN || rope->scaling == OOM_ROPE_LINEAR || rope->scaling == OOM_ROPE_YARN,
                "oom_rope_table: scaling");
    const bool yarn = rope->scaling == OOM_ROPE_YARN;
    OOM_REQUIRE(rope->scaling == OOM_ROPE_PLAIN || (rope->factor >= 1.0 && std::isfinite(rope->factor)),
                "oom_rope_table: factor must be at least 1");
    OOM_REQUIRE(!yarn || (rope->trained_len >= 1 && rope->beta_slow > 0.0 && rope->beta_fast >= rope->beta_slow &&
                          std::isfinite(rope->beta_fast)),
                "oom_rope_table: trained_len must be >= 1 and beta_fast >= beta_slow > 0");
    OOM_REQUIRE(n >= (size_t)rot / 2, "oom_rope_table: table smaller than rot_dim / 2");
    const double two_pi = 6.283185307179586476925286766559;
    double lo = 0, hi = 0;
    if (yarn) {
        // the dim whose pair makes `beta` turns over the trained length
        const auto dim = [&](double beta) {
            return rot * std::log((double)rope->trained_len / (two_pi * beta)) / (2.0 * std::log(rope->base));
        };
        lo = std::fmax(0.0, std::floor(dim(rope->beta_fast)));
        hi = std::fmin(rot - 1.0, std::ceil(dim(rope->beta_slow)));
    }
    for (int i = 0; i < rot / 2; i++) {
        double f = std::pow(rope->base, -2.0 * i / rot);
        if (rope->scaling == OOM_ROPE_LINEAR) f /= rope->factor;
        if (yarn) {
            const double r = std::fmin(1.0, std::fmax(0.0, (i - lo) / std::fmax(hi - lo, 0.001)));
            f = f * (1.0 - r) + f / rope->factor * r;
        }
        turns[i] = (uint64_t)std::nearbyint(std::ldexp(f / two_pi, 64));  // f <= 1: below 2^62
    }
    *magnitude = yarn ? (float)(0.1 * std::log(rope->factor) + 1.0) : 1.0f;
    return OOM_OK;
}

namespace oom {

static int rope_checks(const char* what, const RopeArgs& a, int layout, int x_dtype, int out_dtype) {
    const std::string w = what;
    OOM_REQUIRE(a.d >= 8 && a.d % 8 == 0 && a.d <= 1024, w + ": head_dim must be a multiple of 8 up to 1024");
    OOM_REQUIRE(a.rot >= 2 && a.rot % 2 == 0 && a.rot <= a.d, w + ": rot_dim must be even, at most head_dim");
    OOM_REQUIRE(layout == OOM_ROPE_HALF || layout == OOM_ROPE_INTERLEAVED, w + ": layout");
    OOM_REQUIRE(x_dtype == OOM_F32 || x_dtype == OOM_BF16, w + ": x_dtype");
    OOM_REQUIRE(out_dtype == OOM_F32 || out_dtype == OOM_BF16, w + ": out_dtype");
    OOM_REQUIRE(a.T >= 0 && a.H >= 1 && a.H <= 4096, w + ": T must be >= 0, heads 1 to 4096");
    OOM_REQUIRE(std::isfinite(a.magnitude), w + ": magnitude must be finite");
    OOM_REQUIRE(a.q_stride >= (int64_t)a.H * a.d && a.out_stride >= (int64_t)a.H * a.d && a.q_stride % 8 == 0 &&
                    a.out_stride % 8 == 0,
                w + ": strides must be multiples of 8 elements, at least a token's heads");
    if (a.T == 0) return OOM_OK;
    OOM_REQUIRE(a.q && a.out && a.positions && a.turns, w + ": null buffer");
    OOM_REQUIRE(aligned(a.q, 16) && aligned(a.out, 16) && aligned(a.turns, 8),
                w + ": buffers of heads must be 16-byte aligned");
    return OOM_OK;
}

template <bool APPEND>
static int launch_rope(const char* what, const RopeArgs& a, int layout, int x_dtype, int out_dtype, hipStream_t st) {
    const int64_t elems = (int64_t)(a.H + (APPEND ? 2 * a.Hkv : 0)) * (a.d / 2);
    for (int64_t t0 = 0; t0 < a.T; t0 += 65535) {
        RopeArgs b = a;
        const int n = (int)std::min<int64_t>(65535, a.T - t0);
        const int64_t xb = x_dtype == OOM_BF16 ? 2 : 4, ob = out_dtype == OOM_BF16 ? 2 : 4;
        b.q = (const uint8_t*)a.q + t0 * a.q_stride * xb;
        b.out = (uint8_t*)a.out + t0 * a.out_stride * ob;
        b.positions += t0;
        if (APPEND) {
            b.k = (const uint8_t*)a.k + t0 * a.k_stride * xb;
            b.v = (const uint8_t*)a.v + t0 * a.v_stride * xb;
            b.slots += t0;
        }
        const dim3 grid((uint32_t)cdiv(elems, 256), n), block(256);
        if (x_dtype == OOM_BF16 && out_dtype == OOM_BF16)
            hipLaunchKernelGGL((rope_kernel<OOM_BF16, OOM_BF16, APPEND>), grid, block, 0, st, b, layout);
        else if (x_dtype == OOM_BF16)
            hipLaunchKernelGGL((rope_kernel<OOM_BF16, OOM_F32, APPEND>), grid, block, 0, st, b, layout);
        else if (out_dtype == OOM_BF16)
            hipLaunchKernelGGL((rope_kernel<OOM_F32, OOM_BF16, APPEND>), grid, block, 0, st, b, layout);
        else
            hipLaunchKernelGGL((rope_kernel<OOM_F32, OOM_F32, APPEND>), grid, block, 0, st, b, layout);
        if (int rc = launched(what)) return rc;
    }
    return OOM_OK;
}

}  // namespace oom

extern "C" int oom_rope(const void* x, int x_dtype, int64_t x_stride, const int32_t* positions, const uint64_t* turns,
                        int rot_dim, int layout, float magnitude, int inverse, void* out, int out_dtype,
                        int64_t out_stride, int T, int heads, int d, void* stream) {
    using namespace oom;
    RopeArgs a = {};
    a.q = x;
    a.q_stride = x_stride;
    a.positions = positions;
    a.turns = turns;
    a.rot = rot_dim;
    a.d = d;
    a.T = T;
    a.H = heads;
    a.magnitude = magnitude;
    a.sign = inverse ? -1.0f : 1.0f;
    a.out = out;
    a.out_stride = out_stride;
    if (int rc = rope_checks("oom_rope", a, layout, x_dtype, out_dtype)) return rc;
    return launch_rope<false>("oom_rope", a, layout, x_dtype, out_dtype, as_stream(stream));
}

extern "C" int oom_rope_append_paged(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                     int64_t v_stride, int x_dtype, const int32_t* positions, const int64_t* slots,
                                     const uint64_t* turns, int rot_dim, int layout, float magnitude, void* q_out,
                                     int out_dtype, int64_t out_stride, uint16_t* k_pages, uint16_t* v_pages,
                                     int n_pages, int page_size, int T, int heads, int kv_heads, int d, void* stream) {
    using namespace oom;
    RopeArgs a = {};
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.positions = positions;
    a.slots = slots;
    a.turns = turns;
    a.rot = rot_dim;
    a.d = d;
    a.T = T;
    a.H = heads;
    a.Hkv = kv_heads;
    a.magnitude = magnitude;
    a.sign = 1.0f;
    a.out = q_out;
    a.out_stride = out_stride;
    a.kp = k_pages;
    a.vp = v_pages;
    a.page_size = page_size;
    a.n_slots = (int64_t)n_pages * page_size;
    if (int rc = rope_checks("oom_rope_append_paged", a, layout, x_dtype, out_dtype)) return rc;
    OOM_REQUIRE(kv_heads >= 1 && kv_heads <= 4096, "oom_rope_append_paged: kv_heads must be 1 to 4096");
    OOM_REQUIRE(n_pages >= 1 && page_size >= 16 && page_size % 16 == 0,
                "oom_rope_append_paged: n_pages must be >= 1 and page_size a multiple of 16");
    OOM_REQUIRE(k_stride >= (int64_t)kv_heads * d && v_stride >= (int64_t)kv_heads * d && k_stride % 8 == 0 &&
                    v_stride % 8 == 0,
                "oom_rope_append_paged: strides must be multiples of 8 elements, at least a token's heads");
    if (T == 0) return OOM_OK;
    OOM_REQUIRE(k && v && slots && k_pages && v_pages, "oom_rope_append_paged: null buffer");
    OOM_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(k_pages, 16) && aligned(v_pages, 16),
                "oom_rope_append_paged: buffers of heads must be 16-byte aligned");
    return launch_rope<true>("oom_rope_append_paged", a, layout, x_dtype, out_dtype, as_stream(stream));
}
