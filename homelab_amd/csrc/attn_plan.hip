// The attention plan of one step's batch, made once on the device and used by every layer:
// the tiles of 128 packed query rows of each sequence with the keys that they see, split over
// the keys where there are too few of them to fill the chip, longest first (blocks start in
// order, so the short ones fill the gaps at the end). Also the new tokens' positions and
// cache slots, which the rotary and append kernels take.
#include "common.hpp"

namespace oom {

struct PlanArgs {
    const int32_t* cu_q;
    const int32_t* kv_lens;  // null: prompts, whose keys are their own tokens
    const int32_t* table;
    int max_pages, n_pages, page_size, B, T, G, Hkv;
    int64_t max_items, max_merge_rows, max_part_rows;
    int32_t* positions;
    int64_t* slots;
    int32_t* plan;
};

struct PlanSeq {
    int q0, n, kv;
};
// Sequence b as the plan takes it: its tokens within [0, T), its keys within its pages.
__device__ __forceinline__ PlanSeq plan_seq(const PlanArgs& a, int b) {
    PlanSeq s;
    s.q0 = min(max(a.cu_q[b], 0), a.T);
    s.n = min(max(a.cu_q[b + 1], s.q0), a.T) - s.q0;
    s.kv = s.n;
    if (a.kv_lens) s.kv = (int)min((int64_t)max(a.kv_lens[b], 0), (int64_t)a.max_pages * a.page_size);
    return s;
}

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_BUCKETS = 256;

// Tile t's sequence and its row range and keys; rows 0 where cu_q does not rise and the tile falls
// outside its sequence.
struct PlanTile {
    int b, q0, row0, rows, off, keys, nkt;
};
__device__ __forceinline__ PlanTile plan_tile(const PlanArgs& a, const int* pre, int t) {
    int lo = 0, hi = a.B;  // pre[lo] <= t < pre[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= t) lo = mid;
        else hi = mid;
    }
    const PlanSeq s = plan_seq(a, lo);
    PlanTile p;
    p.b = lo;
    p.q0 = s.q0;
    const int64_t row0 = (int64_t)(t - pre[lo]) * ATTN_ROWS, rows = (int64_t)s.n * a.G - row0;
    p.row0 = (int)row0;
    p.rows = row0 < 0 || rows < 0 ? 0 : (int)min((int64_t)ATTN_ROWS, rows);
    p.off = s.kv - s.n;
    p.keys = max(0, p.off + (p.row0 + p.rows - 1) / a.G + 1);
    p.nkt = (p.keys + ATTN_KEYS - 1) / ATTN_KEYS;
    return p;
}

// Exclusive prefix sums of v over the block's threads; `total` the whole.
__device__ int block_scan(int v, int* tmp, int& total) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int x = v;
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) tmp[wave] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < PLAN_THREADS / 64; w++) {
        if (w < wave) before += tmp[w];
        total += tmp[w];
    }
    return before + x - v;
}

// Block 0 writes the items; the blocks after it the positions and slots of 1024 tokens each.
__global__ void __launch_bounds__(PLAN_THREADS) attn_plan_kernel(PlanArgs a) {
    const int tid = threadIdx.x;
    if (blockIdx.x > 0) {
        const int t = (int)(blockIdx.x - 1) * PLAN_THREADS + tid;
        if (t >= a.T) return;
        int lo = 0, hi = a.B;  // the last sequence that starts at or before t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu_q[mid] <= t) lo = mid;
            else hi = mid;
        }
        PlanSeq s = {0, 0, 0};
        if (a.B > 0) s = plan_seq(a, lo);
        const bool in = t >= s.q0 && t < s.q0 + s.n;
        const int pos = in ? s.kv - s.n + (t - s.q0) : 0;
        if (a.positions) a.positions[t] = pos;
        if (a.slots) {
            int64_t slot = -1;
            if (in && pos >= 0 && a.table) {
                const int page = a.table[(size_t)lo * a.max_pages + pos / a.page_size];
                if (page >= 0 && page < a.n_pages) slot = (int64_t)page * a.page_size + pos % a.page_size;
            }
            a.slots[t] = slot;
        }
        return;
    }
    __shared__ int pre[ATTN_MAXB + 1], tmp[PLAN_THREADS / 64], hist[PLAN_BUCKETS];
    __shared__ unsigned long long work;
    __shared__ int longest, n_parts, n_merges;
    constexpr int PER = ATTN_MAXB / PLAN_THREADS;
    int mine[PER], sum = 0, tiles;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int b = tid * PER + i;
        mine[i] = 0;
        if (b < a.B) mine[i] = (int)(((int64_t)plan_seq(a, b).n * a.G + ATTN_ROWS - 1) / ATTN_ROWS);
        sum += mine[i];
    }
    if (tid == 0) {
        work = 0;
        longest = 1;
        n_parts = n_merges = 0;
        pre[0] = 0;
    }
    if (tid < PLAN_BUCKETS) hist[tid] = 0;
    int at = block_scan(sum, tmp, tiles);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        at += mine[i];
        pre[tid * PER + i + 1] = at;
    }
    __syncthreads();
    // a batch whose cu_q does not rise can claim more rows than there are: what the plan has no
    // room for is left out
    tiles = (int)min((int64_t)tiles, a.max_items);
    unsigned long long w = 0;
    int most = 1;
    for (int t = tid; t < tiles; t += PLAN_THREADS) {
        const PlanTile p = plan_tile(a, pre, t);
        if (p.rows == 0) continue;
        w += p.nkt;
        most = max(most, p.nkt);
    }
    atomicAdd(&work, w);
    atomicMax(&longest, most);
    __syncthreads();
    // prompts are not split: their rows alone fill the chip, or their keys are few
    int ks = longest;
    if (a.kv_lens) {
        const unsigned long long k = (work * a.Hkv + ATTN_SPLIT_BLOCKS - 1) / ATTN_SPLIT_BLOCKS;
        ks = (int)min((unsigned long long)longest, max(k, 4ull));
    }
    const auto bucket = [&](int n) { return PLAN_BUCKETS - 1 - (int)((int64_t)n * (PLAN_BUCKETS - 1) / ks); };
    for (int t = tid; t < tiles; t += PLAN_THREADS) {
        const PlanTile p = plan_tile(a, pre, t);
        if (p.rows == 0) continue;
        const int n = p.nkt, ns = max(1, (n + ks - 1) / ks);
        if (ns > 1) atomicAdd(&hist[0], ns - 1);
        atomicAdd(&hist[bucket(n - (ns - 1) * ks)], 1);
    }
    __syncthreads();
    int items;
    const int h = tid < PLAN_BUCKETS ? hist[tid] : 0;
    const int first = block_scan(h, tmp, items);
    if (tid < PLAN_BUCKETS) hist[tid] = first;
    __syncthreads();
    int32_t* const list = a.plan + ATTN_PLAN_HEAD;
    int4* const merges = reinterpret_cast<int4*>(list + a.max_items * ATTN_ITEM_WORDS);
    for (int t = tid; t < tiles; t += PLAN_THREADS) {
        const PlanTile p = plan_tile(a, pre, t);
        if (p.rows == 0) continue;
        const int ns = max(1, (p.nkt + ks - 1) / ks);
        int part = -1;
        if (ns > 1) {
            part = atomicAdd(&n_parts, ns * p.rows);
            const int m = atomicAdd(&n_merges, p.rows);
            if (part + (int64_t)ns * p.rows > a.max_part_rows || m + (int64_t)p.rows > a.max_merge_rows) continue;
            // a row to merge: its token, its head of the group (bit 30: it sees no key), its first
            // partial, and how many there are, p.rows apart
            for (int r = 0; r < p.rows; r++) {
                const int tok = (p.row0 + r) / a.G, g = p.row0 + r - tok * a.G;
                merges[m + r] = make_int4(p.q0 + tok, g | (p.off + tok < 0 ? 1 << 30 : 0), part + r, ns | p.rows << 16);
            }
        }
        for (int i = 0; i < ns; i++) {
            const int k0 = i * ks * ATTN_KEYS, k1 = min(p.keys, k0 + ks * ATTN_KEYS);
            const int at = atomicAdd(&hist[i + 1 < ns ? 0 : bucket(p.nkt - (ns - 1) * ks)], 1);
            if (at >= a.max_items) continue;
            int32_t* e = list + (int64_t)at * ATTN_ITEM_WORDS;
            *reinterpret_cast<int4*>(e) = make_int4(p.q0, p.row0, p.rows, p.off);
            *reinterpret_cast<int4*>(e + 4) = make_int4(k0, k1, ns > 1 ? part + i * p.rows : -1, p.b);
        }
    }
    __syncthreads();
    if (tid == 0) {
        a.plan[ATTN_PLAN_ITEMS] = (int)min((int64_t)items, a.max_items);
        a.plan[ATTN_PLAN_MERGES] = (int)min((int64_t)n_merges, a.max_merge_rows);
    }
}

}  // namespace oom

extern "C" size_t oom_attn_plan_size(int T, int B, int heads, int kv_heads, int d) {
    if (T < 0 || B < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || d < 1) return 0;
    return (size_t)oom::attn_plan_dims(T, B, heads, kv_heads).words;
}

extern "C" int oom_attn_plan(const int32_t* cu_q, const int32_t* kv_lens, const int32_t* page_table, int max_pages,
                             int n_pages, int page_size, int T, int B, int heads, int kv_heads, int d,
                             int32_t* positions, int64_t* slots, int32_t* plan, void* stream) {
    using namespace oom;
    OOM_REQUIRE(d == 64 || d == 128 || d == 256, "oom_attn_plan: head_dim must be 64, 128 or 256");
    OOM_REQUIRE(kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && heads <= 4096,
                "oom_attn_plan: heads must be a multiple of kv_heads, at most 4096");
    OOM_REQUIRE(T >= 0 && B >= 0 && B <= ATTN_MAXB && (int64_t)T * heads < (1ll << 31),
                "oom_attn_plan: at most 4096 sequences, and fewer than 2^31 rows of heads");
    OOM_REQUIRE((kv_lens == nullptr) == (page_table == nullptr), "oom_attn_plan: kv_lens and page_table go together");
    if (page_table) {
        OOM_REQUIRE(page_size >= 16 && page_size % 16 == 0, "oom_attn_plan: page_size must be a multiple of 16");
        OOM_REQUIRE(n_pages >= 1 && max_pages >= 1 && (int64_t)max_pages * page_size <= ATTN_MAX_KEYS,
                    "oom_attn_plan: n_pages and max_pages must be >= 1, a sequence at most 128 Mi keys");
    }
    OOM_REQUIRE(page_table || !slots, "oom_attn_plan: slots need a page_table");
    OOM_REQUIRE(plan && cu_q, "oom_attn_plan: null buffer");
    OOM_REQUIRE(aligned(plan, 16), "oom_attn_plan: plan must be 16-byte aligned");
    const AttnPlanDims p = attn_plan_dims(T, B, heads, kv_heads);
    PlanArgs a;
    a.cu_q = cu_q;
    a.kv_lens = kv_lens;
    a.table = page_table;
    a.max_pages = max_pages;
    a.n_pages = n_pages;
    a.page_size = page_size;
    a.B = B;
    a.T = T;
    a.G = heads / kv_heads;
    a.Hkv = kv_heads;
    a.max_items = p.items;
    a.max_merge_rows = p.merge_rows;
    a.max_part_rows = p.part_rows;
    a.positions = positions;
    a.slots = slots;
    a.plan = plan;
    const int blocks = 1 + (positions || slots ? (int)cdiv(T, PLAN_THREADS) : 0);
    hipLaunchKernelGGL(attn_plan_kernel, dim3(blocks), dim3(PLAN_THREADS), 0, as_stream(stream), a);
    return launched("oom_attn_plan");
}
