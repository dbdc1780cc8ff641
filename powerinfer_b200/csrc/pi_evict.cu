// Eviction from the KV cache in 8 bits: a sequence of len slots is cut to `keep` by the attention weight that its slots have accumulated.
//
// Kept are the first n_sink slots, the last n_recent, and of the others those with the largest weights, the lowest slots among equals.  A kept
// slot below `keep` stays where it is; the kept ones behind it, in ascending order, take the places of the evicted ones below it, in
// ascending order.  So nothing moves that need not, no row is both read and written, and a block is written by one warp.  Attention does not ask
// for the order of slots.  A block's scale becomes the largest of the scales of the rows that are in it now, and codes of other scales
// rne(code * (scale / that)).
//
// k_evict_select, a CTA per sequence and KV head: the weights as ordered integers in shared memory, the threshold bit by bit
// from counts (a histogram's atomics meet in the few exponents that weights have), then bit maps of what is above it and of what equals it, and sums over
// their words.  k_evict_move, a warp per block: rows are gathered and scaled.  Bound by latency: the bytes are those of the weights and of the moved rows.
#include "pi_kv_q8.cuh"

namespace pi {

static constexpr int EV_THREADS = 1024, EV_WARPS = EV_THREADS / 32;
static constexpr int EV_CACHED = 36864;                               // weights that shared memory holds beside the maps of 262144 slots

// order of weights as unsigned numbers: -0 as 0, what is not a number above all others
__device__ __forceinline__ uint32_t ev_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
// sum of v over the CTA, for everybody (s_red: EV_WARPS words, free again at the next call's barrier)
__device__ __forceinline__ int ev_sum(int v, int * s_red) {
    const int w = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = w;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, s_red[threadIdx.x & 31]);
}
// sum of v over the threads before this one
__device__ __forceinline__ int ev_before(int v, int * s_red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += x; }
    __syncthreads();
    if (lane == 31) s_red[warp] = incl;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; w++) before += s_red[w];
    return before + incl - v;
}

__global__ void __launch_bounds__(EV_THREADS) k_evict_select(const EvictArgs p, int cached) {
    extern __shared__ uint32_t ev_smem[];
    __shared__ int s_red[EV_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = blockIdx.x, i = blockIdx.y, n_ctx = p.c.n_ctx, words_max = (n_ctx + 31) / 32;
    uint32_t * above = ev_smem, * equal = above + words_max;         // bit maps of the slots; later: kept ones, and sums of holes before each word
    uint32_t * keys = equal + words_max;
    pdl_launch();
    pdl_wait();
    int32_t * kept = p.kept + ((size_t)i * p.c.H + h) * p.keep;
    const int sq = p.seq ? p.seq[i] : i;
    bool dead = sq < 0 || sq >= p.c.n_seq;
    if (p.seq) {                                                      // of entries that name one sequence the last one counts
        bool later = false;
        for (int j = i + 1 + tid; j < p.n; j += EV_THREADS) later |= p.seq[j] == sq;
        dead |= __syncthreads_or(later) != 0;
    }
    const int len = dead ? 0 : max(0, min(p.len[i], n_ctx));
    const size_t row = ((size_t)max(0, dead ? 0 : sq) * p.c.H + h) * n_ctx;
    const float * w = p.w + row;
    float * w_out = p.w_out ? p.w_out + row : nullptr;
    if (len <= p.keep) {                                              // nothing to evict
        for (int j = tid; j < p.keep; j += EV_THREADS) {
            kept[j] = j < len ? j : -1;
            if (w_out && j < len) w_out[j] = w[j];
        }
        return;
    }
    // ---- candidates: slots c0 .. c1 - 1, of which `need` stay
    const int c0 = p.n_sink, c1 = len - p.n_recent, need = p.keep - p.n_sink - p.n_recent, n_c = c1 - c0;
    const bool here = n_c <= cached;
    uint32_t most = 0u, least = 0xffffffffu;
    for (int j = tid; j < n_c; j += EV_THREADS) {
        const uint32_t k = ev_key(w[c0 + j]);
        if (here) keys[j] = k;
        most = max(most, k); least = min(least, k);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    __shared__ uint32_t s_most[EV_WARPS], s_least[EV_WARPS];
    if (lane == 0) { s_most[warp] = most; s_least[warp] = least; }
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, s_most[lane]);
    least = __reduce_min_sync(0xffffffffu, s_least[lane]);
    auto key = [&](int j) { return here ? keys[j] : ev_key(__ldcg(w + c0 + j)); };
    // ---- the need-th largest key: its bits from the first one in which keys differ, each from a count of the keys that have it
    uint32_t t = most;
    int greater = 0;                                                  // keys above t
    if (need > 0 && most != least) {
        const int top = 31 - __clz(most ^ least);
        t = top == 31 ? 0u : most >> (top + 1) << (top + 1);
        for (int bit = top; bit >= 0; bit--) {
            const uint32_t want = t >> bit | 1u;
            int n = 0;
            if (here) {
#pragma unroll 4
                for (int j = tid; j < n_c; j += EV_THREADS) n += keys[j] >> bit == want;
            } else {
#pragma unroll 4
                for (int j = tid; j < n_c; j += EV_THREADS) n += key(j) >> bit == want;
            }
            n = ev_sum(n, s_red);
            if (greater + n >= need) t |= 1u << bit; else greater += n;
        }
    }
    // ---- bit maps over the slots
    const int words = (len + 31) / 32;
    for (int x = warp; x < words; x += EV_WARPS) {
        const int j = x * 32 + lane;
        bool a = false, e = false;
        if (j < len) {
            if (j < c0 || j >= c1) a = true;
            else if (need > 0) { const uint32_t k = key(j - c0); a = k > t; e = k == t; }
        }
        const uint32_t am = __ballot_sync(0xffffffffu, a), em = __ballot_sync(0xffffffffu, e);
        if (lane == 0) { above[x] = am; equal[x] = em; }
    }
    __syncthreads();
    // ---- of the equals the first ones
    const int per = (words + EV_THREADS - 1) / EV_THREADS, x0 = min(tid * per, words), x1 = min(x0 + per, words);
    int mine = 0;
    for (int x = x0; x < x1; x++) mine += __popc(equal[x]);
    int left = need - greater - ev_before(mine, s_red);
    for (int x = x0; x < x1; x++) {
        uint32_t e = equal[x], take = e;
        const int n = __popc(e);
        if (n > left) { take = 0u; for (int k = 0; k < left; k++) { const uint32_t b = e & -e; take |= b; e ^= b; } }
        left = max(0, left - n);
        above[x] |= take;
    }
    // ---- holes below the budget: their number before each word
    const int keep_words = (p.keep + 31) / 32;
    auto below = [&](int x) { return x * 32 + 32 <= p.keep ? 0xffffffffu : x * 32 >= p.keep ? 0u : (1u << (p.keep - x * 32)) - 1u; };
    __syncthreads();
    int holes = 0, movers = 0;
    for (int x = x0; x < x1; x++) { const uint32_t m = below(x); holes += __popc(~above[x] & m); movers += __popc(above[x] & ~m); }
    int before_h = ev_before(holes, s_red), before_m = ev_before(movers, s_red);
    for (int x = x0; x < x1; x++) { equal[x] = before_h; before_h += __popc(~above[x] & below(x)); }
    __syncthreads();
    // ---- who takes which place
    for (int x = x0; x < x1; x++) {
        uint32_t m = above[x] & ~below(x);
        while (m) {
            const int j = x * 32 + __ffs(m) - 1;
            m &= m - 1;
            int lo = 0, hi = keep_words - 1;                          // the last word with at most before_m holes before it
            while (lo < hi) { const int mid = (lo + hi + 1) / 2; if ((int)equal[mid] <= before_m) lo = mid; else hi = mid - 1; }
            uint32_t e = ~above[lo] & below(lo);
            for (int k = before_m - (int)equal[lo]; k > 0; k--) e &= e - 1;
            kept[lo * 32 + __ffs(e) - 1] = j;
            before_m++;
        }
    }
    for (int x = warp; x < keep_words; x += EV_WARPS) {
        const int j = x * 32 + lane;
        if (j < p.keep && (above[x] >> lane & 1u)) kept[j] = j;
    }
    if (!w_out) return;
    __syncthreads();                                                  // (this CTA's writes to kept are visible to it)
    for (int j = tid; j < p.keep; j += EV_THREADS) w_out[j] = w[kept[j]];
}

__device__ __forceinline__ uint32_t ev_scale(uint32_t c, float ratio) {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) r |= (uint32_t)(__float2int_rn((float)(int8_t)(c >> (8 * j)) * ratio) & 255) << (8 * j);
    return r;
}

static constexpr int MV_THREADS = 256;

__global__ void __launch_bounds__(MV_THREADS) k_evict_move(const EvictArgs p) {
    const int lane = threadIdx.x & 31, B = p.c.block, blocks = p.keep >> p.c.shift;
    pdl_launch();
    pdl_wait();
    const int64_t unit = (int64_t)blockIdx.x * (MV_THREADS / 32) + (threadIdx.x >> 5);       // (keys or values, head, block)
    if (unit >= (int64_t)2 * p.c.H * blocks) return;
    const int b = (int)(unit % blocks), hv = (int)(unit / blocks), h = hv >> 1, which = hv & 1, i = blockIdx.y;
    const int sq = p.seq ? p.seq[i] : i;
    if (sq < 0 || sq >= p.c.n_seq) return;
    const int32_t * kept = p.kept + ((size_t)i * p.c.H + h) * p.keep + b * B;
    int src[4]; bool moves = false;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int r = u * 32 + lane;
        src[u] = r < B ? __ldcg(kept + r) : -1;
        moves |= src[u] >= p.keep;
    }
    if (!__any_sync(0xffffffffu, moves)) return;
    const size_t head = (size_t)sq * p.c.H + h;
    float * scale = (which ? p.c.vs : p.c.ks) + head * (p.c.n_ctx >> p.c.shift);
    float of[4], now = 0.f;
#pragma unroll
    for (int u = 0; u < 4; u++) { of[u] = src[u] >= 0 ? scale[src[u] >> p.c.shift] : 0.f; now = fmaxf(now, of[u]); }
    now = warp_max(now);
    const float old = scale[b];
    int8_t * codes = (which ? p.c.v : p.c.k) + head * p.c.n_ctx * p.c.hd;
    const int hd = p.c.hd, per_row = hd / 16, n16 = B * per_row;
    __syncwarp();
    if (lane == 0 && now != old) scale[b] = now;
    for (int e0 = 0; e0 < n16; e0 += 128) {
        uint4 c[4]; float ratio[4]; int64_t to[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int e = e0 + u * 32 + lane, r = min(e / per_row, B - 1), piece = e - r * per_row;
            int from = -1; float s = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int f = __shfl_sync(0xffffffffu, src[k], r & 31); const float o = __shfl_sync(0xffffffffu, of[k], r & 31);
                if (r >> 5 == k) { from = f; s = o; }
            }
            to[u] = -1;
            // (a row that stays is written where the block's steps grew; behind the sequence's end nothing is)
            if (e < n16 && from >= 0 && (from != b * B + r || now != s)) {
                to[u] = ((int64_t)b * B + r) * hd + piece * 16;
                ratio[u] = s == now ? 1.f : s / now;
                c[u] = *reinterpret_cast<const uint4 *>(codes + (size_t)from * hd + piece * 16);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (to[u] >= 0)
                *reinterpret_cast<uint4 *>(codes + to[u]) = make_uint4(ev_scale(c[u].x, ratio[u]), ev_scale(c[u].y, ratio[u]), ev_scale(c[u].z, ratio[u]), ev_scale(c[u].w, ratio[u]));
    }
}

int launch_kv_evict_q8(const EvictArgs & a, cudaStream_t st) {
    const int words = (a.c.n_ctx + 31) / 32, cached = a.c.n_ctx < EV_CACHED ? a.c.n_ctx : EV_CACHED;
    const size_t smem = (size_t)words * 8 + (size_t)cached * 4;
    static bool done[16] = {false};
    int dev = 0;
    PI_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16 || !done[dev]) {
        PI_CUDA(cudaFuncSetAttribute(k_evict_select, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
        if (dev >= 0 && dev < 16) done[dev] = true;
    }
    PI_CUDA(launch_k(k_evict_select, dim3(a.c.H, a.n), dim3(EV_THREADS), smem, st, true, a, cached));
    const int64_t units = (int64_t)2 * a.c.H * (a.keep >> a.c.shift);
    PI_CUDA(launch_k(k_evict_move, dim3((unsigned)((units + MV_THREADS / 32 - 1) / (MV_THREADS / 32)), a.n), dim3(MV_THREADS), 0, st, true, a));
    return PI_OK;
}

}  // namespace pi
