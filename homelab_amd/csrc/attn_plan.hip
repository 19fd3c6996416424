// The attention plan of one step's batch, made once on the device and used by every layer:
// the tiles of 128 packed query rows of each sequence with the keys that they see, split over
// the keys where there are too few of them to fill the chip, longest first (blocks start in
// order, so the short ones fill the gaps at the end); sequences of at most 32 rows over a paged cache
// in a list of their own (attn_few.hpp). Also the new tokens' positions and
// cache slots, which the rotary and append kernels take.
#include "common.hpp"

namespace oom {

struct PlanArgs {
    const int32_t* cu_q;
    const int32_t* kv_lens;  // null: prompts, whose keys are their own tokens
    const int32_t* table;
    int max_pages, n_pages, page_size, B, T, G, Hkv, few_rows, split_blocks, sign;
    int64_t max_items, max_few, max_merge_rows;
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

// A tile of rows with its keys; rows 0 where cu_q does not rise and the tile falls outside its
// sequence. few: the sequence's only tile, its keys in units of ATTN_FEW_KEYS.
struct PlanTile {
    int b, q0, row0, rows, off, keys, unit, n;
    bool few;
};

// Block 0 writes the items; the blocks after it the positions and slots of 1024 tokens each.
__global__ void __launch_bounds__(PLAN_THREADS) attn_plan_kernel(PlanArgs a) {
    const int tid = threadIdx.x, lane = tid & 63;
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
    __shared__ int pre[ATTN_MAXB + 1], seq_q0[ATTN_MAXB], seq_n[ATTN_MAXB], seq_kv[ATTN_MAXB];
    __shared__ int tmp[PLAN_THREADS / 64], hist[2][PLAN_BUCKETS];
    __shared__ unsigned long long work[2];
    __shared__ int longest[2], n_parts, n_merges;
    constexpr int PER = ATTN_MAXB / PLAN_THREADS;
    for (int b = tid; b < a.B; b += PLAN_THREADS) {
        const PlanSeq s = plan_seq(a, b);
        seq_q0[b] = s.q0;
        seq_n[b] = s.n;
        seq_kv[b] = s.kv;
    }
    if (tid < 2) {
        work[tid] = 0;
        longest[tid] = 1;
    }
    if (tid == 0) n_parts = n_merges = pre[0] = 0;
    if (tid < 2 * PLAN_BUCKETS) (&hist[0][0])[tid] = 0;
    __syncthreads();
    int mine[PER], sum = 0, tiles;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int b = tid * PER + i;
        mine[i] = b < a.B ? (int)(((int64_t)seq_n[b] * a.G + ATTN_ROWS - 1) / ATTN_ROWS) : 0;
        sum += mine[i];
    }
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
    const auto tile = [&](int t) {
        int lo = 0, hi = a.B;  // pre[lo] <= t < pre[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= t) lo = mid;
            else hi = mid;
        }
        PlanTile p;
        p.b = lo;
        p.q0 = seq_q0[lo];
        const int64_t all = (int64_t)seq_n[lo] * a.G, row0 = (int64_t)(t - pre[lo]) * ATTN_ROWS, rows = all - row0;
        p.row0 = (int)row0;
        p.rows = row0 < 0 || rows < 0 ? 0 : (int)min((int64_t)ATTN_ROWS, rows);
        p.off = seq_kv[lo] - seq_n[lo];
        p.keys = max(0, p.off + (p.row0 + p.rows - 1) / a.G + 1);
        p.few = a.kv_lens && all <= a.few_rows;
        p.unit = p.few ? ATTN_FEW_KEYS : ATTN_KEYS;
        p.n = (p.keys + p.unit - 1) / p.unit;
        return p;
    };
    for (int t = tid; t < tiles; t += PLAN_THREADS) {
        const PlanTile p = tile(t);
        if (p.rows == 0) continue;
        atomicAdd(&work[p.few], (unsigned long long)p.n);
        atomicMax(&longest[p.few], p.n);
    }
    __syncthreads();
    // Units a split. Prompts are not split: their rows alone fill the chip, or their keys are few. Else
    // the work's even share a block, or up to a half more where that keeps the splits to as many
    // blocks as run at once, so that no few of them make a second round (512 tokens over 16 Ki
    // keys, d 128: 284 us with the share, 275 so; over 8000 keys at d 256: 148 with a quarter more at
    // most, 135 so; with no bound, 3 x 300 tokens over up to 3000 keys at d 256 took 104 us, not 71).
    int ks[2] = {longest[0], longest[1]};
    if (a.kv_lens) {
        PlanTile p = {};
        if (tid < tiles) p = tile(tid);
        for (int f = 0; f < 2; f++) {
            const int slots = f ? ATTN_FEW_BLOCKS : a.split_blocks;
            const unsigned long long even = (work[f] * a.Hkv + slots - 1) / slots;
            const int share = (int)min((unsigned long long)longest[f], max(even, f ? 1ull : 4ull));
            ks[f] = share;
            // (more tiles than threads are more than the blocks: no search)
            if (tiles > PLAN_THREADS) continue;
            for (int k = share; k <= share + share / 2 && k < longest[f]; k += max(1, share / 16)) {
                int all;
                block_scan(p.rows > 0 && p.few == (f == 1) ? (p.n + k - 1) / k : 0, tmp, all);
                if ((int64_t)all * a.Hkv <= slots) {
                    ks[f] = k;
                    break;
                }
            }
        }
    }
    const auto splits = [&](const PlanTile& p) { return max(1, (p.n + ks[p.few] - 1) / ks[p.few]); };
    const auto bucket = [&](const PlanTile& p, int n) {
        return PLAN_BUCKETS - 1 - (int)((int64_t)n * (PLAN_BUCKETS - 1) / ks[p.few]);
    };
    for (int t = tid; t < tiles; t += PLAN_THREADS) {
        const PlanTile p = tile(t);
        if (p.rows == 0) continue;
        const int ns = splits(p);
        if (ns > 1) atomicAdd(&hist[p.few][0], ns - 1);
        atomicAdd(&hist[p.few][bucket(p, p.n - (ns - 1) * ks[p.few])], 1);
    }
    __syncthreads();
    int items[2];
    for (int f = 0; f < 2; f++) {
        const int h = tid < PLAN_BUCKETS ? hist[f][tid] : 0;
        const int first = block_scan(h, tmp, items[f]);
        if (tid < PLAN_BUCKETS) hist[f][tid] = first;
        __syncthreads();
    }
    int32_t* const list = a.plan + ATTN_PLAN_HEAD;
    int32_t* const few_list = list + a.max_items * ATTN_ITEM_WORDS;
    int4* const merges = reinterpret_cast<int4*>(few_list + a.max_few * ATTN_ITEM_WORDS);
    // tile p's split i
    const auto put = [&](const PlanTile& p, int i, int ns, int part) {
        const int len = ks[p.few] * p.unit;
        const int at = atomicAdd(&hist[p.few][i + 1 < ns ? 0 : bucket(p, p.n - (ns - 1) * ks[p.few])], 1);
        if (at >= (p.few ? a.max_few : a.max_items)) return;
        int4* e = reinterpret_cast<int4*>((p.few ? few_list : list) + (int64_t)at * ATTN_ITEM_WORDS);
        e[0] = make_int4(p.q0, p.row0, p.rows, p.off);
        e[1] = make_int4(i * len, min(p.keys, (i + 1) * len), ns > 1 ? part + i * p.rows : -1, p.b);
    };
    for (int t0 = tid - lane; t0 < tiles; t0 += PLAN_THREADS) {
        const int t = t0 + lane;
        PlanTile p = {};
        if (t < tiles) p = tile(t);
        const int ns = p.rows > 0 ? splits(p) : 0;
        if (ns == 1) put(p, 0, 1, -1);
        // split tiles one after the other, the wave's lanes on their items and their rows to merge
        for (unsigned long long left = __ballot(ns > 1); left; left &= left - 1) {
            const int from = __builtin_ctzll(left);
            PlanTile s;
            s.b = __shfl(p.b, from);
            s.q0 = __shfl(p.q0, from);
            s.row0 = __shfl(p.row0, from);
            s.rows = __shfl(p.rows, from);
            s.off = __shfl(p.off, from);
            s.keys = __shfl(p.keys, from);
            s.unit = __shfl(p.unit, from);
            s.n = __shfl(p.n, from);
            s.few = __shfl((int)p.few, from) != 0;
            const int n = __shfl(ns, from);
            int part = 0, m = 0;
            if (lane == 0) {
                part = atomicAdd(&n_parts, n * s.rows);
                m = atomicAdd(&n_merges, s.rows);
            }
            part = __shfl(part, 0);
            m = __shfl(m, 0);
            // a row to merge: its token, its head of the group (bit 30: it sees no key), its first
            // partial, and how many there are, s.rows apart. (The partials fit whatever cu_q holds, since
            // their bound follows from the split; rows to merge are more than there is room for
            // only where sequences overlap.)
            for (int r = lane; r < s.rows && m + (int64_t)r < a.max_merge_rows; r += 64) {
                const int tok = (s.row0 + r) / a.G, g = s.row0 + r - tok * a.G;
                merges[m + r] = make_int4(s.q0 + tok, g | (s.off + tok < 0 ? 1 << 30 : 0), part + r, n | s.rows << 16);
            }
            for (int i = lane; i < n; i += 64) put(s, i, n, part);
        }
    }
    __syncthreads();
    if (tid == 0) {
        a.plan[ATTN_PLAN_SIGN] = a.sign;
        a.plan[ATTN_PLAN_ITEMS] = (int)min((int64_t)items[0], a.max_items);
        a.plan[ATTN_PLAN_FEW] = (int)min((int64_t)items[1], a.max_few);
        a.plan[ATTN_PLAN_SPLIT] = (int)min((int64_t)ks[0] * ATTN_KEYS, (int64_t)INT32_MAX);
        a.plan[ATTN_PLAN_MERGES] = (int)min((int64_t)n_merges, a.max_merge_rows);
    }
}

}  // namespace oom

extern "C" size_t oom_attn_plan_size(int T, int B, int heads, int kv_heads, int d) {
    if (T < 0 || B < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || d < 1) return 0;
    return (size_t)oom::attn_plan_dims(T, B, heads, kv_heads, d).words;
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
    const AttnPlanDims p = attn_plan_dims(T, B, heads, kv_heads, d);
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
    a.few_rows = attn_has_few(T, B, a.G, d) ? attn_few_rows(d) : 0;
    a.split_blocks = attn_split_blocks(d);
    a.sign = attn_plan_sign(T, B, heads, kv_heads, d, page_table ? max_pages : 0, page_table ? page_size : 0);
    a.max_items = p.items;
    a.max_few = p.few_items;
    a.max_merge_rows = p.merge_rows;
    a.positions = positions;
    a.slots = slots;
    a.plan = plan;
    const int blocks = 1 + (positions || slots ? (int)cdiv(T, PLAN_THREADS) : 0);
    hipLaunchKernelGGL(attn_plan_kernel, dim3(blocks), dim3(PLAN_THREADS), 0, as_stream(stream), a);
    return launched("oom_attn_plan");
}
