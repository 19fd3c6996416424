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

typedef __bf16 rbf16x2 __attribute__((ext_vector_type(2)));
typedef float rf32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t r_pack(float a, float b) {
    const rf32x2 f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, rbf16x2));  // RNE
}

__device__ __forceinline__ void turn_sincos(int pos, uint64_t f, float& s, float& c) {
    const int64_t t = (int64_t)((uint64_t)(int64_t)pos * f);  // turns * 2^64, in [-1/2, 1/2)
    const float half_turns = (float)(int32_t)(t >> 32) * 0x1p-31f;  // angle / pi in [-1, 1), 2^-32 turns off at most
    sincospif(half_turns, &s, &c);
}

// V consecutive elements, 16 bytes of an fp32 run of 4 or a bf16 run of 8 (the other type's in two
// halves or one).
template <int DT, int V>
__device__ __forceinline__ void load_run(const void* p, int64_t i, float (&x)[V]) {
    if constexpr (DT == OOM_BF16) {
        uint32_t w[V / 2];
        if constexpr (V == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
            w[0] = v.x, w[1] = v.y;
        }
#pragma unroll
        for (int e = 0; e < V / 2; e++) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    } else {
        const float4* f = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
        for (int e = 0; e < V / 4; e++) {
            const float4 v = f[e];
            x[4 * e] = v.x, x[4 * e + 1] = v.y, x[4 * e + 2] = v.z, x[4 * e + 3] = v.w;
        }
    }
}
template <int DT, int V>
__device__ __forceinline__ void store_run(void* p, int64_t i, const float (&x)[V]) {
    if constexpr (DT == OOM_BF16) {
        uint32_t w[V / 2];
#pragma unroll
        for (int e = 0; e < V / 2; e++) w[e] = r_pack(x[2 * e], x[2 * e + 1]);
        uint16_t* o = reinterpret_cast<uint16_t*>(p) + i;
        if constexpr (V == 8) *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
    } else {
        float4* f = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
#pragma unroll
        for (int e = 0; e < V / 4; e++) f[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
    }
}

constexpr int ROPE_TABLE = 2048;  // cosines and sines a block holds

// Two runs of V elements of a head a thread: a unit. With rot a multiple of 2 V, unit u under rot /
// 2 V is dims V u .. and their partners rot / 2 further (halves), or dims 2 V u .. (interleaved);
// the units after it dims 2 V u .. as they are (one run where d ends). The cosines and sines of a
// token are the same for every head: a block computes them once, a thread each, into LDS while its
// first elements arrive. (Each thread its unit's own, with no barrier to wait at: 32.8 against
// 24.9 us for 2047 fp32 tokens of 28 heads, 4.4 against 4.1 for 64 bf16 tokens of 80.)
template <int XDT, int ODT, int V, int LAYOUT, bool APPEND>
__global__ void __launch_bounds__(256) rope_units_kernel(RopeArgs a, int units, int step, int tokens) {
    __shared__ __align__(16) float2 cs[ROPE_TABLE];
    const int half = a.rot / 2, turned = a.rot / (2 * V);
    const int t0 = (int)blockIdx.y * tokens, own = (int)(threadIdx.x / (uint32_t)(units * step)), t = t0 + own;
    const int in = (int)(threadIdx.x % (uint32_t)(units * step)), u = in % units;
    const bool live = own < tokens && t < a.T;
    const int heads = a.H + (APPEND ? 2 * a.Hkv : 0);
    const int i = u < turned && LAYOUT == OOM_ROPE_HALF ? V * u : 2 * V * u;
    const int j = u < turned && LAYOUT == OOM_ROPE_HALF ? i + half : i + V;
    const bool two = j < a.d;
    int64_t slot = -1, row = 0;
    if constexpr (APPEND) {
        if (live) slot = a.slots[t];
        if (slot >= 0 && slot < a.n_slots)
            row = slot / a.page_size * a.Hkv * a.page_size + slot % a.page_size;  // of KV head 0
        else slot = -1;
    }
    float p[V], q[V] = {};
    const auto load = [&](int hd) {
        const bool is_k = APPEND && hd >= a.H, is_v = APPEND && hd >= a.H + a.Hkv;
        if (is_k && slot < 0) return;
        const void* x = is_v ? a.v : is_k ? a.k : a.q;
        const int64_t at = is_v   ? t * a.v_stride + (int64_t)(hd - a.H - a.Hkv) * a.d
                           : is_k ? t * a.k_stride + (int64_t)(hd - a.H) * a.d
                                  : t * a.q_stride + (int64_t)hd * a.d;
        load_run<XDT, V>(x, at + i, p);
        if (two) load_run<XDT, V>(x, at + j, q);
    };
    int hd = (int)blockIdx.x * step + in / units;
    if (live && hd < heads) load(hd);
    for (int e = threadIdx.x; e < min(tokens, a.T - t0) * half; e += 256) {
        float sn, co;
        turn_sincos(a.positions[t0 + e / half], a.turns[e % half], sn, co);
        cs[e] = make_float2(co * a.magnitude, sn * (a.sign * a.magnitude));
    }
    __syncthreads();
    if (!live) return;
    float c[V], s[V];
    if (u < turned) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const float4 v = *reinterpret_cast<const float4*>(cs + own * half + V * u + e);
            c[e] = v.x, s[e] = v.y, c[e + 1] = v.z, s[e + 1] = v.w;
        }
    }
    while (hd < heads) {
        const bool is_k = APPEND && hd >= a.H, is_v = APPEND && hd >= a.H + a.Hkv;
        if (u < turned && !is_v) {
            if constexpr (LAYOUT == OOM_ROPE_HALF) {
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float y = p[e], z = q[e];
                    p[e] = fmaf(y, c[e], -(z * s[e]));
                    q[e] = fmaf(y, s[e], z * c[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V / 2; e++) {
                    const float y = p[2 * e], z = p[2 * e + 1], v = q[2 * e], w = q[2 * e + 1];
                    p[2 * e] = fmaf(y, c[e], -(z * s[e]));
                    p[2 * e + 1] = fmaf(y, s[e], z * c[e]);
                    q[2 * e] = fmaf(v, c[e + V / 2], -(w * s[e + V / 2]));
                    q[2 * e + 1] = fmaf(v, s[e + V / 2], w * c[e + V / 2]);
                }
            }
        }
        if (!is_k) {
            const int64_t to = t * a.out_stride + (int64_t)hd * a.d;
            store_run<ODT, V>(a.out, to + i, p);
            if (two) store_run<ODT, V>(a.out, to + j, q);
        } else if (slot >= 0) {
            const int g = is_v ? hd - a.H - a.Hkv : hd - a.H;
            uint16_t* out = (is_v ? a.vp : a.kp) + (row + (int64_t)g * a.page_size) * a.d;
            store_run<OOM_BF16, V>(out, i, p);
            if (two) store_run<OOM_BF16, V>(out, j, q);
        }
        hd += (int)gridDim.x * step;
        if (hd < heads) load(hd);
    }
}

// One thread a pair (or two elements past rot) of the queries, then of the keys, then of the
// values: for a rot that is no multiple of two runs. Reading both before writing either, it may work in
// place (as does the other kernel).
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
    const auto w = [what](const char* msg) { return std::string(what) + msg; };
    OOM_REQUIRE(a.d >= 8 && a.d % 8 == 0 && a.d <= 1024, w(": head_dim must be a multiple of 8 up to 1024"));
    OOM_REQUIRE(a.rot >= 2 && a.rot % 2 == 0 && a.rot <= a.d, w(": rot_dim must be even, at most head_dim"));
    OOM_REQUIRE(layout == OOM_ROPE_HALF || layout == OOM_ROPE_INTERLEAVED, w(": layout"));
    OOM_REQUIRE(x_dtype == OOM_F32 || x_dtype == OOM_BF16, w(": x_dtype"));
    OOM_REQUIRE(out_dtype == OOM_F32 || out_dtype == OOM_BF16, w(": out_dtype"));
    OOM_REQUIRE(a.T >= 0 && a.H >= 1 && a.H <= 4096, w(": T must be >= 0, heads 1 to 4096"));
    OOM_REQUIRE(std::isfinite(a.magnitude), w(": magnitude must be finite"));
    OOM_REQUIRE(a.q_stride >= (int64_t)a.H * a.d && a.out_stride >= (int64_t)a.H * a.d && a.q_stride % 8 == 0 &&
                    a.out_stride % 8 == 0,
                w(": strides must be multiples of 8 elements, at least a token's heads"));
    if (a.T == 0) return OOM_OK;
    OOM_REQUIRE(a.q && a.out && a.positions && a.turns, w(": null buffer"));
    OOM_REQUIRE(aligned(a.q, 16) && aligned(a.out, 16) && aligned(a.turns, 8),
                w(": buffers of heads must be 16-byte aligned"));
    return OOM_OK;
}

// The launch of units: a block holds `tokens` tokens' units of `step` heads each, 256 threads at most,
// and walks over the heads, or gridDim.x blocks share them. Enough blocks to fill the chip
// come from the tokens alone in a long prompt, which leaves a thread several heads of its
// unit; few tokens spread their heads over more blocks.
template <int XDT, int ODT, bool APPEND>
static void launch_rope_t(const RopeArgs& a, int layout, hipStream_t st) {
    constexpr int V = XDT == OOM_BF16 ? 8 : 4;
    const int units = a.rot / (2 * V) + (int)cdiv(a.d - a.rot, 2 * V), heads = a.H + (APPEND ? 2 * a.Hkv : 0);
    if (a.rot % (2 * V) != 0) {
        const int64_t pairs = (int64_t)heads * (a.d / 2);
        hipLaunchKernelGGL((rope_kernel<XDT, ODT, APPEND>), dim3((uint32_t)cdiv(pairs, 256), (uint32_t)a.T), dim3(256), 0, st,
                           a, layout);
        return;
    }
    const int step = std::max(1, std::min(256 / units, heads));
    int tokens = std::max(1, std::min(256 / (units * step), 2 * ROPE_TABLE / a.rot));
    tokens = (int)std::min<int64_t>(tokens, cdiv(a.T, 1024));
    const int64_t rows = cdiv(a.T, tokens);
    const int64_t share = std::min<int64_t>(cdiv(heads, step), std::max<int64_t>(1, cdiv(1024, rows)));
    const dim3 grid((uint32_t)share, (uint32_t)rows), block(256);
    if (layout == OOM_ROPE_HALF)
        hipLaunchKernelGGL((rope_units_kernel<XDT, ODT, V, OOM_ROPE_HALF, APPEND>), grid, block, 0, st, a, units, step, tokens);
    else
        hipLaunchKernelGGL((rope_units_kernel<XDT, ODT, V, OOM_ROPE_INTERLEAVED, APPEND>), grid, block, 0, st, a, units, step,
                           tokens);
}

template <bool APPEND>
static int launch_rope(const char* what, const RopeArgs& a, int layout, int x_dtype, int out_dtype, hipStream_t st) {
    for (int64_t t0 = 0; t0 < a.T; t0 += 65535) {  // grid.y
        RopeArgs b = a;
        b.T = (int)std::min<int64_t>(65535, a.T - t0);
        const int64_t xb = x_dtype == OOM_BF16 ? 2 : 4, ob = out_dtype == OOM_BF16 ? 2 : 4;
        b.q = (const uint8_t*)a.q + t0 * a.q_stride * xb;
        b.out = (uint8_t*)a.out + t0 * a.out_stride * ob;
        b.positions += t0;
        if (APPEND) {
            b.k = (const uint8_t*)a.k + t0 * a.k_stride * xb;
            b.v = (const uint8_t*)a.v + t0 * a.v_stride * xb;
            b.slots += t0;
        }
        if (x_dtype == OOM_BF16 && out_dtype == OOM_BF16) launch_rope_t<OOM_BF16, OOM_BF16, APPEND>(b, layout, st);
        else if (x_dtype == OOM_BF16) launch_rope_t<OOM_BF16, OOM_F32, APPEND>(b, layout, st);
        else if (out_dtype == OOM_BF16) launch_rope_t<OOM_F32, OOM_BF16, APPEND>(b, layout, st);
        else launch_rope_t<OOM_F32, OOM_F32, APPEND>(b, layout, st);
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
