// Trees of drafted tokens: the masks and positions that the parents stand for, and the path that a target model agrees with.
//
//     A(t) = {t} + A(parent(t))     pos(t) = pos0 + |A(t)| - 1          next of c on the path: the lowest u with parent(u) = c, tokens(u) = choice(c)
//
// A parent's number is smaller than its child's, so ancestors come in descending order: one walk to the root makes a row's words one after the other.  The
// next token of every one is found at once (the lowest child that agrees, by minima in shared memory); the path is then a chain of loads from there.
// Bound by the launch and by the longest chain of dependent loads from shared memory, 30 clocks each; bytes and operations are next to none.  Both kernels together: a tree of 25 tokens 4.8 us, 64 of up to 192 7.3.
#include "pi_kv_paged.cuh"

namespace pi {

static constexpr int TREE_THREADS = 128;

__global__ void __launch_bounds__(TREE_THREADS) k_tree_mask(const RaggedB b, const int32_t * parents, uint64_t * mask, int words, int32_t * pos) {
    extern __shared__ int s_parent[];
    const int i = blockIdx.y, tid = threadIdx.x, t = blockIdx.x * TREE_THREADS + tid;
    pdl_launch();
    pdl_wait();
    const int2 e = entry_rows(b, i);
    const int upto = min(e.y, (int)(blockIdx.x + 1) * TREE_THREADS);  // (ancestors have smaller numbers)
    for (int u = tid; u < upto; u += TREE_THREADS) s_parent[u] = parents[e.x + u];
    __syncthreads();
    if (t >= e.y) return;
    uint64_t * row = mask + (size_t)(e.x + t) * words;
    int at = words - 1, depth = -1;
    uint64_t word = 0;
    for (int u = t, before = t + 1; (unsigned)u < (unsigned)before; before = u, u = s_parent[u]) {      // (a parent that is not before its child is none)
        const int w = u >> 6;
        depth++;
        if (w >= words) continue;
        for (; at > w; at--) { row[at] = word; word = 0; }
        word |= 1ull << (u & 63);
    }
    for (; at >= 0; at--) { row[at] = word; word = 0; }
    if (pos) pos[e.x + t] = b.pos0[i] + depth;
}

__global__ void __launch_bounds__(TREE_THREADS) k_tree_accept(const RaggedB b, int width, const int32_t * tokens, const int32_t * parents, const int32_t * choice, int32_t * path,
                                                              int32_t * n_path, int32_t * next) {
    extern __shared__ int s_next[];
    __shared__ int s_n;
    const int i = blockIdx.x, tid = threadIdx.x;
    pdl_launch();
    pdl_wait();
    const int2 e = entry_rows(b, i);
    constexpr int NONE = 0x7fffffff;
    for (int u = tid; u < e.y; u += TREE_THREADS) s_next[u] = NONE;
    __syncthreads();
    for (int u = tid; u < e.y; u += TREE_THREADS) {
        const int c = parents[e.x + u];
        if (c >= 0 && c < u && tokens[e.x + u] == choice[e.x + c]) atomicMin(s_next + c, u);
    }
    __syncthreads();
    int32_t * row = path + (size_t)i * width;
    if (tid == 0) {
        int n = 0, last = -1;
        for (int u = e.y > 0 ? 0 : NONE; u != NONE; u = s_next[u]) { row[n++] = u; last = u; }      // (numbers rise: at most e.y steps)
        n_path[i] = n;
        next[i] = last < 0 ? -1 : choice[e.x + last];
        s_n = n;
    }
    __syncthreads();
    for (int r = s_n + tid; r < width; r += TREE_THREADS) row[r] = -1;
}

int launch_tree_mask(const RaggedB & b, const int32_t * parents, uint64_t * mask, int words, int32_t * pos, cudaStream_t st) {
    PI_CUDA(launch_k(k_tree_mask, dim3((unsigned)((b.max_new + TREE_THREADS - 1) / TREE_THREADS), b.n), dim3(TREE_THREADS), (size_t)b.max_new * 4, st, true, b, parents, mask, words, pos));
    return PI_OK;
}
int launch_tree_accept(const RaggedB & b, int width, const int32_t * tokens, const int32_t * parents, const int32_t * choice, int32_t * path, int32_t * n_path, int32_t * next, cudaStream_t st) {
    PI_CUDA(launch_k(k_tree_accept, dim3(b.n), dim3(TREE_THREADS), (size_t)b.max_new * 4, st, true, b, width, tokens, parents, choice, path, n_path, next));
    return PI_OK;
}

}  // namespace pi
