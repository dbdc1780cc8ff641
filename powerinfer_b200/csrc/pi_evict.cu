// Eviction from the KV cache in 8 bits: a sequence of len slots is cut to `keep` by the attention weight that its slots have accumulated.
//
// Kept are the first n_sink slots, the last n_recent, and of the others those with the largest weights, the lowest slots among equals.  A kept
// slot below `keep` stays where it is; the kept ones behind it, in ascending order, take the places of the evicted ones below it, in
// ascending order.  So nothing moves that need not, no row is both read and written, and a block is written by one warp.  Attention does not ask
// for the order of slots.  A block's scale becomes the largest of the scales of the rows that are in it now, and codes of other scales
// rne(code * (scale / that)).
//
// k_evict_select, a CTA per sequence and KV head: the weights as ordered integers in registers, EV_REGS a thread (longer sequences: that many at a time, read
// again); the threshold from three histograms of 11, 11 and 10 bits (whole numbers: their order does not matter); then bit maps of what is above it and of
// what equals it, sums over their words, and the holes' slots as a list from which every mover takes its place.  k_evict_move, a warp per block: rows are gathered
// and scaled.  Few heads: bound by the instructions that one SM issues for a head's slots.  (A cluster of eight SMs a head was slower: the histograms travel.)
// Many: by the bytes of the moved rows.  Measured: 16384 slots to 2048, 8 heads: 21 us and 10 us; 1280 to 1024, 16 sequences of 32 heads: 19 us and 30 us.
// (Four copies of the first histogram, against lanes that meet in a bin: the same 21 us.)
#include "pi_kv_q8.cuh"

namespace pi {

static constexpr int EV_THREADS = 1024, EV_REGS = 16;                 // threads at most
static constexpr int EV_LIST = 16384;                                 // holes that the list holds at a time
static constexpr int EV_BINS = 2048;

// order of weights as unsigned numbers: -0 as 0, what is not a number above all others; 0 is no weight's
__device__ __forceinline__ uint32_t ev_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
// sum of v over the threads before this one (s_red: 32 words)
__device__ __forceinline__ int ev_before(int v, int * s_red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += x; }
    __syncthreads();
    if (lane == 31) s_red[warp] = incl;
    __syncthreads();
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? s_red[lane] : 0);
    return before + incl - v;
}

__global__ void __launch_bounds__(EV_THREADS) k_evict_select(const EvictArgs p, int listed) {
    extern __shared__ uint32_t ev_smem[];
    __shared__ int s_red[32];
    __shared__ __align__(16) int s_bin[EV_BINS];
    __shared__ int s_found[2];
    const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5, CHUNK = EV_REGS * nt;
    const int h = blockIdx.x, i = blockIdx.y, n_ctx = p.c.n_ctx, words_max = (n_ctx + 31) / 32;
    uint32_t * above = ev_smem, * equal = above + words_max;         // bit maps of the slots
    int * list = (int *)(equal + words_max);                          // the holes' slots
    pdl_launch();
    pdl_wait();
    int32_t * kept = p.kept + ((size_t)i * p.c.H + h) * p.keep;
    const int sq = p.seq ? p.seq[i] : i;
    bool dead = sq < 0 || sq >= p.c.n_seq;
    if (p.seq) {                                                      // of entries that name one sequence the last one counts
        bool later = false;
        for (int j = i + 1 + tid; j < p.n; j += nt) later |= p.seq[j] == sq;
        dead |= __syncthreads_or(later) != 0;
    }
    const int len = dead ? 0 : max(0, min(p.len[i], n_ctx));
    const size_t row = ((size_t)max(0, dead ? 0 : sq) * p.c.H + h) * n_ctx;
    const float * w = p.w + row;
    float * w_out = p.w_out ? p.w_out + row : nullptr;
    if (len <= p.keep) {                                              // nothing to evict
        for (int j = tid; j < p.keep; j += nt) {
            kept[j] = j < len ? j : -1;
            if (w_out && j < len) w_out[j] = w[j];
        }
        return;
    }
    // ---- candidates: slots c0 .. c1 - 1, of which `need` stay.  Others have the key 0.
    const int c0 = p.n_sink, c1 = len - p.n_recent;
    int need = p.keep - p.n_sink - p.n_recent, have = -1;
    uint32_t key[EV_REGS];                                            // of the slots have + u * nt + tid
    auto load = [&](int from) {
        if (from == have) return;
        have = from;
        float x[EV_REGS];
#pragma unroll
        for (int u = 0; u < EV_REGS; u++) { const int j = from + u * nt + tid; x[u] = j >= c0 && j < c1 ? __ldcg(w + j) : 0.f; }
#pragma unroll
        for (int u = 0; u < EV_REGS; u++) { const int j = from + u * nt + tid; key[u] = j >= c0 && j < c1 ? ev_key(x[u]) : 0u; }
    };
    // ---- t, the need-th largest key, and how many of those that equal it stay
    uint32_t t = 0xffffffffu;
    if (need > 0) {
        t = 0u;
#pragma unroll 1
        for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1) {
            const int bins = shift ? EV_BINS : 1024, hi = shift == 21 ? 32 : shift == 10 ? 21 : 10;       // bits shift .. hi - 1
            for (int x = tid; x < EV_BINS; x += nt) s_bin[x] = 0;
            __syncthreads();
            for (int from = 0; from < len; from += CHUNK) {
                load(from);
#pragma unroll
                for (int u = 0; u < EV_REGS; u++) {
                    const uint32_t k = key[u];
                    if (k != 0u && (hi == 32 || k >> hi == t >> hi)) atomicAdd(&s_bin[k >> shift & (uint32_t)(bins - 1)], 1);
                }
            }
            __syncthreads();
            // thread x has the x-th bins from above: the bin in which the need-th key lies
            const int per = bins / nt, b0 = bins - 1 - tid * per;
            int mine = 0;
            for (int x = 0; x < per; x++) mine += s_bin[b0 - x];
            int before = ev_before(mine, s_red);
            if (before < need && need <= before + mine)
                for (int x = 0; x < per; x++) {
                    const int c = s_bin[b0 - x];
                    if (before < need && need <= before + c) { s_found[0] = b0 - x; s_found[1] = need - before; }
                    before += c;
                }
            __syncthreads();
            t |= (uint32_t)s_found[0] << shift;
            need = s_found[1];
        }
    }
    // ---- bit maps over the slots
    const int words = (len + 31) / 32;
    for (int from = 0; from < len; from += CHUNK) {
        load(from);
#pragma unroll
        for (int u = 0; u < EV_REGS; u++) {
            const int k = (from + u * nt + tid) >> 5;
            const uint32_t am = __ballot_sync(0xffffffffu, key[u] > t), em = __ballot_sync(0xffffffffu, key[u] == t);      // (t is never 0)
            if (lane == 0 && k < words) { above[k] = am; equal[k] = em; }
        }
    }
    __syncthreads();
    // slots of word k that are below `end`
    auto under = [&](int k, int end) { return k * 32 + 32 <= end ? 0xffffffffu : k * 32 >= end ? 0u : (1u << (end - k * 32)) - 1u; };
    // ---- of the equals the first ones; then `equal` takes the number of holes (below the budget) or movers (behind it) before each word
    const int per = (words + nt - 1) / nt, x0 = min(tid * per, words), x1 = min(x0 + per, words);
    int mine = 0;
    for (int x = x0; x < x1; x++) mine += __popc(equal[x]);
    int left = need - ev_before(mine, s_red);
    for (int x = x0; x < x1; x++) {
        uint32_t e = equal[x], take = e;
        const int n = __popc(e);
        if (n > left) { take = 0u; for (int k = 0; k < left; k++) { const uint32_t b = e & (0u - e); take |= b; e ^= b; } }
        left = max(0, left - n);
        above[x] |= take | under(x, c0) | (under(x, len) & ~under(x, c1));
    }
    const int keep_words = (p.keep + 31) / 32;
    auto below = [&](int x) { return under(x, p.keep); };
    int holes = 0, movers = 0;
    for (int x = x0; x < x1; x++) { const uint32_t m = below(x); holes += __popc(~above[x] & m); movers += __popc(above[x] & ~m); }
    int before_h = ev_before(holes, s_red), before_m = ev_before(movers, s_red);
    // (a word with both, where the budget ends inside it: its holes' number; its movers are the first ones)
    for (int x = x0; x < x1; x++) {
        const uint32_t m = below(x);
        equal[x] = m ? before_h : before_m;
        before_h += __popc(~above[x] & m);
        before_m += __popc(above[x] & ~m);
    }
    // ---- who takes which place: the holes of ranks `first` and on as a list, from which the movers of the same ranks read
    __syncthreads();
    for (int first = 0; first < p.keep; first += listed) {
        for (int k = warp; k < keep_words; k += warps) {
            const uint32_t m = below(k), e = ~above[k] & m;
            const int rank = (int)equal[k] + __popc(e & ((1u << lane) - 1u)) - first, j = k * 32 + lane;
            if (e >> lane & 1u) { if (rank >= 0 && rank < listed) list[rank] = j; }
            else if (first == 0 && m >> lane & 1u) kept[j] = j;
        }
        __syncthreads();
        for (int kb = p.keep / 32 + warp; kb < words; kb += 8 * warps) {
            int to[8]; float v[8];                                    // (eight words' weights on their way; nothing behind the budget is written)
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int k = kb + u * warps;
                to[u] = -1;
                if (k >= words) continue;
                const uint32_t m = below(k), e = above[k] & ~m;
                const int rank = (m ? 0 : (int)equal[k]) + __popc(e & ((1u << lane) - 1u)) - first;
                if ((e >> lane & 1u) && rank >= 0 && rank < listed) {
                    to[u] = list[rank];
                    if (w_out) v[u] = __ldcg(w + k * 32 + lane);
                }
            }
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (to[u] >= 0) {
                    kept[to[u]] = (kb + u * warps) * 32 + lane;
                    if (w_out) w_out[to[u]] = v[u];
                }
        }
        __syncthreads();
    }
    if (w_out && w_out != w)
        for (int kb = warp; kb < keep_words; kb += 8 * warps) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) { const int j = (kb + u * warps) * 32 + lane; if (j < p.keep) v[u] = __ldcg(w + j); }
#pragma unroll
            for (int u = 0; u < 8; u++) { const int j = (kb + u * warps) * 32 + lane; if (j < p.keep && above[j >> 5] >> lane & 1u) w_out[j] = v[u]; }
        }
}

// Four codes times ratio, rounded to the nearest whole number.  Whole numbers become FP32 and back by their place in the mantissa (2^23 + 128 + code; the
// product + 1.5 x 2^23): conversions run at an eighth of the rate of sums, and half of the kernel was them.
__device__ __forceinline__ uint32_t ev_scale(uint32_t c, float ratio) {
    const uint32_t u = c ^ 0x80808080u;
    uint32_t r[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float f = __fsub_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 + j)), 8388736.f);
        r[j] = __float_as_uint(__fadd_rn(__fmul_rn(f, ratio), 12582912.f));
    }
    return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
}

static constexpr int MV_THREADS = 256, MV_U = 4;                      // pieces of 16 codes on their way, a lane

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
    int row = lane / per_row, part = lane - row * per_row;            // of a lane's next piece; 32 pieces on
    const int row_on = 32 / per_row, part_on = 32 - row_on * per_row;
    for (int e0 = 0; e0 < n16; e0 += MV_U * 32) {
        uint4 c[MV_U]; float ratio[MV_U]; int to[MV_U];
#pragma unroll
        for (int u = 0; u < MV_U; u++) {
            const int r = min(row, B - 1), piece = part;
            const bool in = row < B;
            row += row_on; part += part_on;
            if (part >= per_row) { part -= per_row; row++; }
            int from = -1; float s = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (k * 32 >= B) break;
                const int f = __shfl_sync(0xffffffffu, src[k], r & 31); const float o = __shfl_sync(0xffffffffu, of[k], r & 31);
                if (r >> 5 == k) { from = f; s = o; }
            }
            to[u] = -1;
            // (a row that stays is written where the block's steps grew; behind the sequence's end nothing is)
            if (in && from >= 0 && (from != b * B + r || now != s)) {
                to[u] = r * hd + piece * 16;
                ratio[u] = s == now ? 1.f : s / now;
                c[u] = *reinterpret_cast<const uint4 *>(codes + (size_t)from * hd + piece * 16);
            }
        }
#pragma unroll
        for (int u = 0; u < MV_U; u++)
            if (to[u] >= 0)
                *reinterpret_cast<uint4 *>(codes + (size_t)b * B * hd + to[u]) = make_uint4(ev_scale(c[u].x, ratio[u]), ev_scale(c[u].y, ratio[u]), ev_scale(c[u].z, ratio[u]), ev_scale(c[u].w, ratio[u]));
    }
}

int launch_kv_evict_q8(const EvictArgs & a, cudaStream_t st) {
    const int words = (a.c.n_ctx + 31) / 32, listed = a.keep < EV_LIST ? a.keep : EV_LIST;
    const size_t smem = (size_t)words * 8 + (size_t)listed * 4;
    // short sequences: smaller CTAs, of which an SM holds several
    int threads = 128;
    while (threads < EV_THREADS && threads * EV_REGS < a.c.n_ctx) threads *= 2;
    static bool done[16] = {false};
    int dev = 0;
    PI_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16 || !done[dev]) {
        PI_CUDA(cudaFuncSetAttribute(k_evict_select, cudaFuncAttributeMaxDynamicSharedMemorySize, 136 * 1024));
        if (dev >= 0 && dev < 16) done[dev] = true;
    }
    PI_CUDA(launch_k(k_evict_select, dim3(a.c.H, a.n), dim3(threads), smem, st, true, a, listed));
    const int64_t units = (int64_t)2 * a.c.H * (a.keep >> a.c.shift);
    PI_CUDA(launch_k(k_evict_move, dim3((unsigned)((units + MV_THREADS / 32 - 1) / (MV_THREADS / 32)), a.n), dim3(MV_THREADS), 0, st, true, a));
    return PI_OK;
}

}  // namespace pi
