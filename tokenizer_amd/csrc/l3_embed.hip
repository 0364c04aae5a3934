// l3_embed.hip -- embedding lookup and its gradient.
//
//   out[t]  = scale * table[ids[t]]                       (an id outside [0, n_rows): a row of zeros)
//   table[v] (+)= scale * sum over {t : ids[t] = v} of grad[t]
//
// Products and sums are in 32 bits, rounded once where they are stored.
#include "l3_token_kernels.h"

#include "l3_dev.h"

namespace l3 {

namespace {

__device__ __forceinline__ uint64_t ids_that_count(uint64_t n, const uint64_t* n_dev) {
    if (!n_dev) return n;
    const uint64_t m = *n_dev;
    return m < n ? m : n;
}

// Eight columns from `col` on of a row of `dim`.
template <class T>
__device__ __forceinline__ void load_cols(const T* p, uint32_t col, uint32_t dim, float* v) {
    if (col + 8 <= dim) { load8(p + col, v); return; }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = col + i < dim ? (float)p[col + i] : 0.f;
}
template <class T>
__device__ __forceinline__ void store_cols(T* p, uint32_t col, uint32_t dim, const float* v) {
    if (col + 8 <= dim) { store8(p + col, v); return; }
    for (int i = 0; i < 8; i++) if (col + i < dim) p[col + i] = (T)v[i];
}
// ---- lookup -------------------------------------------------------------------------------------------------------
// A thread has kEmbedPer times eight neighbouring columns, all loads in flight before the first store.  What is divided is a
// workgroup's first vector (once) and 32-bit offsets from it.
constexpr int kEmbedThreads = 256, kEmbedPer = 4, kEmbedTile = kEmbedThreads * kEmbedPer;

template <class T, class O>
__global__ __launch_bounds__(kEmbedThreads) void embed_kernel(const int32_t* __restrict__ ids, uint64_t n, const uint64_t* __restrict__ n_dev,
                                                              const T* __restrict__ table, uint32_t rows, uint32_t dim, uint64_t stride,
                                                              O* __restrict__ out, uint64_t out_stride, float scale) {
    const uint32_t per_row = (dim + 7) / 8;
    const uint64_t count = ids_that_count(n, n_dev), total = count * per_row;
    for (uint64_t g0 = (uint64_t)blockIdx.x * kEmbedTile; g0 < total; g0 += (uint64_t)gridDim.x * kEmbedTile) {
        const uint64_t t0 = g0 / per_row;
        const uint32_t r0 = (uint32_t)(g0 - t0 * per_row);
        uint64_t t[kEmbedPer];
        uint32_t col[kEmbedPer];
        int32_t id[kEmbedPer];
        float v[kEmbedPer][8];
#pragma unroll
        for (int k = 0; k < kEmbedPer; k++) {
            const uint32_t at = r0 + k * kEmbedThreads + threadIdx.x, row = at / per_row;
            t[k] = t0 + row;
            col[k] = (at - row * per_row) * 8;
            id[k] = t[k] < count ? ids[t[k]] : -1;
        }
#pragma unroll
        for (int k = 0; k < kEmbedPer; k++) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[k][i] = 0.f;
            if (id[k] >= 0 && (uint32_t)id[k] < rows) load_cols(table + (uint64_t)(uint32_t)id[k] * stride, col[k], dim, v[k]);
        }
#pragma unroll
        for (int k = 0; k < kEmbedPer; k++) {
            if (t[k] >= count) continue;
            const bool there = id[k] >= 0 && (uint32_t)id[k] < rows;
#pragma unroll
            for (int i = 0; i < 8; i++) v[k][i] = there ? v[k][i] * scale : 0.f;   // (a row of zeros whatever the scale is)
            store_cols(out + t[k] * out_stride, col[k], dim, v[k]);
        }
    }
}

// ---- gradient: ids sorted -----------------------------------------------------------------------------------------
// Stable counting sort of (id, position) by digits, the lowest first.  An id that is no row, and a position that does not
// count, has the key n_rows and ends up behind all others.  A tile of kSortTile ids per workgroup:
//   sort_count_kernel    how often each digit occurs in the tile
//   sort_place_kernel    adds up the counts of the tiles before it, ranks the tile's ids and writes them to their places
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64, kSortRounds = kSortTile / kSortThreads;
static_assert(kSortThreads == 2 * kSortBins, "two threads a digit add up the tiles' counts");

__device__ __forceinline__ uint32_t sort_key(const int32_t* ids, uint64_t i, uint64_t valid, uint32_t rows) {
    if (i >= valid) return rows;
    const int32_t id = ids[i];
    return id < 0 || (uint32_t)id >= rows ? rows : (uint32_t)id;
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const int32_t* ids, const uint32_t* keys, uint64_t n, const uint64_t* n_dev,
                                                                  uint32_t rows, int shift, uint32_t mask, uint32_t* hist) {
    __shared__ uint32_t cnt[kSortBins];
    if (threadIdx.x < kSortBins) cnt[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t valid = FIRST ? ids_that_count(n, n_dev) : n, lo = (uint64_t)blockIdx.x * kSortTile;
#pragma unroll
    for (int k = 0; k < kSortRounds; k++) {
        const uint64_t i = lo + (uint64_t)k * kSortThreads + threadIdx.x;
        if (i < n) atomicAdd(&cnt[((FIRST ? sort_key(ids, i, valid, rows) : keys[i]) >> shift) & mask], 1u);
    }
    __syncthreads();
    if (threadIdx.x < kSortBins) hist[(uint64_t)blockIdx.x * kSortBins + threadIdx.x] = cnt[threadIdx.x];
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const int32_t* ids, const uint32_t* keys, const uint32_t* poss, uint64_t n,
                                                                  const uint64_t* n_dev, uint32_t rows, int shift, uint32_t mask, int bits,
                                                                  const uint32_t* hist, uint32_t* keys_out, uint32_t* pos_out) {
    __shared__ uint32_t cnt[kSortWaves][kSortBins];
    __shared__ uint32_t half_all[kSortBins], half_before[kSortBins];
    __shared__ uint32_t tmp[kSortWaves];
    const int tid = threadIdx.x, w = wave_id(), lane = lane_id();
    const uint64_t valid = FIRST ? ids_that_count(n, n_dev) : n;
    const uint64_t lo = (uint64_t)blockIdx.x * kSortTile + (uint64_t)w * (kSortTile / kSortWaves);
    uint32_t key[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int k = 0; k < kSortRounds; k++) {
        const uint64_t i = lo + (uint64_t)k * 64 + lane;
        key[k] = i < n ? (FIRST ? sort_key(ids, i, valid, rows) : keys[i]) : 0;
    }
    for (int d = tid; d < kSortWaves * kSortBins; d += kSortThreads) (&cnt[0][0])[d] = 0;
    // where the tile's ids of digit d start: all ids of smaller digits, then those of digit d in the tiles before.  Two threads a
    // digit, every second tile each, eight loads in flight.
    const int digit = tid % kSortBins;
    uint32_t all = 0, before = 0;
    for (uint32_t b0 = tid / kSortBins; b0 < gridDim.x; b0 += 16) {
        uint32_t c[8];
#pragma unroll
        for (int j = 0; j < 8; j++) c[j] = b0 + 2 * j < gridDim.x ? hist[(uint64_t)(b0 + 2 * j) * kSortBins + digit] : 0;
#pragma unroll
        for (int j = 0; j < 8; j++) { all += c[j]; before += b0 + 2 * j < blockIdx.x ? c[j] : 0; }
    }
    if (tid >= kSortBins) { half_all[digit] = all; half_before[digit] = before; }
    __syncthreads();
    if (tid < kSortBins) { all += half_all[digit]; before += half_before[digit]; } else all = 0;
    uint32_t total;
    uint32_t start = block_escan<kSortWaves>(all, tmp, &total) + before;   // (of the first kSortBins threads)
    // ranks: a wave has kSortTile / kSortWaves ids in a row, 64 at a time
#pragma unroll
    for (int k = 0; k < kSortRounds; k++) {
        const bool in = lo + (uint64_t)k * 64 + lane < n;
        const uint32_t d = (key[k] >> shift) & mask;
        u64 same = __ballot(in);
        for (int b = 0; b < bits; b++) {
            const u64 one = __ballot((d >> b) & 1);
            same &= (d >> b) & 1 ? one : ~one;
        }
        // (a lane that has no id takes no part: its `same` may be anything)
        const int first = in ? __builtin_ctzll(same) : 0;
        uint32_t old = 0;
        if (in && lane == first) old = atomicAdd(&cnt[w][d], (uint32_t)__popcll(same));
        old = __shfl(old, first, 64);
        rank[k] = old + (uint32_t)__popcll(same & ((1ull << lane) - 1));
    }
    __syncthreads();
    if (tid < kSortBins) {
        uint32_t c[kSortWaves];
#pragma unroll
        for (int v = 0; v < kSortWaves; v++) c[v] = cnt[v][tid];
#pragma unroll
        for (int v = 0; v < kSortWaves; v++) { cnt[v][tid] = start; start += c[v]; }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortRounds; k++) {
        const uint64_t i = lo + (uint64_t)k * 64 + lane;
        if (i < n) {
            const uint32_t at = cnt[w][(key[k] >> shift) & mask] + rank[k];
            keys_out[at] = key[k];
            pos_out[at] = FIRST ? (uint32_t)i : poss[i];
        }
    }
}

// ---- gradient: runs of one id added up ----------------------------------------------------------------------------
// A walker goes through `chunk` sorted positions for eight columns a thread, in order, four at a time: the four rows of the
// gradient and, where a run of one id ends, the row of the table it is added to are loaded together.  A run that lies inside the
// chunk is stored at once.  A run that crosses a border leaves its part in the workspace: part[2 c] of the run that came in
// from the chunk before, part[2 c + 1] of the run that starts here and goes on; grad_join_kernel adds these up at the chunk
// where the run starts.  Nothing is added by atomics: the same ids give the same bits.
constexpr int kGradThreads = 256, kGradGroup = 4;
constexpr uint32_t kZeroRows = 64;   // rows a workgroup looks after when the gradient is written whole

// lanes of a row, a power of two
inline uint32_t grad_lanes(uint64_t dim) {
    const uint64_t v = (dim + 7) / 8;
    uint32_t l = 1;
    while (l < v && l < (uint32_t)kGradThreads) l *= 2;
    return l;
}

template <class T>
__device__ __forceinline__ void add_scaled(const float* old, const float* sum, float scale, float* v) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = old[i] + scale * sum[i];
}

// Rows [r0, r0 + kZeroRows) of which `named` has no bit become zero; by a whole workgroup.
template <class T>
__device__ __forceinline__ void zero_rows(T* table, uint64_t table_stride, uint64_t rows, uint32_t dim, uint64_t r0, u64 named) {
    static_assert(kZeroRows == 64, "a word of bits");
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const uint32_t per_row = (dim + 7) / 8;
    for (uint32_t j = wave_id(); j < kZeroRows && r0 + j < rows; j += kGradThreads / 64) {
        if ((named >> j) & 1) continue;
        for (uint32_t k = lane_id(); k < per_row; k += 64) store_cols(table + (r0 + j) * table_stride, k * 8, dim, zero);
    }
}

struct GradWalk {
    const uint32_t* keys; const uint32_t* poss; uint64_t n; uint32_t rows;
    uint32_t chunk; uint64_t chunks; uint32_t lanes, col_tiles; uint64_t walk_blocks;
    const void* grad; uint64_t grad_stride; uint32_t dim;
    void* table; uint64_t table_stride;
    float scale; int accumulate;
    float* part; uint64_t dim8;
};

template <class G, class T>
__global__ __launch_bounds__(kGradThreads) void grad_walk_kernel(GradWalk P) {
    const G* __restrict__ grad = (const G*)P.grad;
    T* __restrict__ table = (T*)P.table;
    const uint32_t* __restrict__ keys = P.keys;
    const uint32_t* __restrict__ poss = P.poss;
    const uint32_t rows = P.rows, dim = P.dim;
    if (blockIdx.x >= P.walk_blocks) {   // rows that no id names, when the gradient is written whole: a binary search a row
        const uint64_t r0 = (uint64_t)(blockIdx.x - P.walk_blocks) * kZeroRows;
        const uint32_t r = (uint32_t)r0 + lane_id();
        uint64_t a = 0, b = P.n;
        while (a < b) { const uint64_t m = (a + b) / 2; if (keys[m] < r) a = m + 1; else b = m; }
        zero_rows(table, P.table_stride, rows, dim, r0, __ballot(a < P.n && keys[a] == r));
        return;
    }
    const uint32_t walkers = kGradThreads / P.lanes;
    uint32_t me = threadIdx.x / P.lanes;
    if (P.lanes >= 64) me = (uint32_t)__builtin_amdgcn_readfirstlane((int)me);   // keys and positions are the wave's: scalar loads
    const uint64_t c = (uint64_t)(blockIdx.x / P.col_tiles) * walkers + me;
    const uint32_t col = ((blockIdx.x % P.col_tiles) * P.lanes + threadIdx.x % P.lanes) * 8;
    if (c >= P.chunks || col >= dim) return;
    const uint64_t lo = c * P.chunk, hi = lo + P.chunk < P.n ? lo + P.chunk : P.n;
    if (keys[lo] >= rows) return;
    // the run that came in, if one did
    const uint32_t came_in = lo > 0 && keys[lo - 1] == keys[lo] ? keys[lo] : ~0u;
    float sum[8];
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = 0.f;
    for (uint64_t i = lo; i < hi; i += kGradGroup) {
        uint32_t k[kGradGroup + 1], pos[kGradGroup];
#pragma unroll
        for (int j = 0; j <= kGradGroup; j++) k[j] = i + j < P.n ? keys[i + j] : ~0u;
#pragma unroll
        for (int j = 0; j < kGradGroup; j++) pos[j] = i + j < hi ? poss[i + j] : 0;
        float g[kGradGroup][8], old[kGradGroup][8];
        bool use[kGradGroup], end[kGradGroup];
#pragma unroll
        for (int j = 0; j < kGradGroup; j++) {
            use[j] = i + j < hi && k[j] < rows;
            end[j] = use[j] && k[j + 1] != k[j];
            if (use[j]) load_cols(grad + (uint64_t)pos[j] * P.grad_stride, col, dim, g[j]);
#pragma unroll
            for (int x = 0; x < 8; x++) old[j][x] = 0.f;
            if (end[j] && k[j] != came_in && P.accumulate) load_cols(table + (uint64_t)k[j] * P.table_stride, col, dim, old[j]);
        }
#pragma unroll
        for (int j = 0; j < kGradGroup; j++) {
            if (!use[j]) continue;
#pragma unroll
            for (int x = 0; x < 8; x++) sum[x] += g[j][x];
            if (!end[j]) continue;
            if (k[j] == came_in) {
                store8(P.part + (2 * c) * P.dim8 + col, sum);
            } else {
                float v[8];
                add_scaled<T>(old[j], sum, P.scale, v);
                store_cols(table + (uint64_t)k[j] * P.table_stride, col, dim, v);
            }
#pragma unroll
            for (int x = 0; x < 8; x++) sum[x] = 0.f;
        }
    }
    const uint32_t last = keys[hi - 1];
    if (last < rows && hi < P.n && keys[hi] == last) store8(P.part + (2 * c + (last == came_in ? 0 : 1)) * P.dim8 + col, sum);
}

// Parts of long runs: a workgroup per chunk and 512 columns, every wave a quarter of the parts, four loads in flight.
template <class T>
__global__ __launch_bounds__(kGradThreads) void grad_join_kernel(GradWalk P, uint32_t tiles) {
    __shared__ float acc[kGradThreads / 64 - 1][64][8];
    const uint32_t* __restrict__ keys = P.keys;
    const uint64_t c = blockIdx.x / tiles;
    const uint32_t col = (blockIdx.x % tiles) * 512 + lane_id() * 8;
    const uint64_t lo = c * P.chunk, hi = lo + P.chunk;
    if (hi >= P.n) return;
    const uint32_t k = keys[hi - 1];
    if (k >= P.rows || keys[hi] != k || (lo > 0 && keys[lo - 1] == k)) return;
    uint64_t more = 0;   // chunks behind c that the run comes into
    for (;;) {
        const uint64_t d = c + 1 + more + lane_id();
        const u64 m = __ballot(d < P.chunks && keys[d * P.chunk] == k);
        if (m == ~0ull) { more += 64; continue; }
        more += (uint64_t)__builtin_ctzll(~m);
        break;
    }
    const int w = wave_id();
    T* row = (T*)P.table + (uint64_t)k * P.table_stride;
    const bool in = col < P.dim;
    float sum[8], old[8];
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = old[i] = 0.f;
    if (in) {
        if (w == 0) {
            if (P.accumulate) load_cols(row, col, P.dim, old);
            load8(P.part + (2 * c + 1) * P.dim8 + col, sum);
        }
        const uint64_t d1 = c + 1 + more * (w + 1) / 4;
        for (uint64_t d = c + 1 + more * w / 4; d < d1; d += 4) {
            float v[4][8];
#pragma unroll
            for (int j = 0; j < 4; j++) if (d + j < d1) load8(P.part + 2 * (d + j) * P.dim8 + col, v[j]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (d + j < d1) {
#pragma unroll
                    for (int i = 0; i < 8; i++) sum[i] += v[j][i];
                }
            }
        }
    }
    if (w) {
#pragma unroll
        for (int i = 0; i < 8; i++) acc[w - 1][lane_id()][i] = sum[i];
    }
    __syncthreads();
    if (w || !in) return;
    for (int x = 0; x < kGradThreads / 64 - 1; x++) {
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] += acc[x][lane_id()][i];
    }
    float v[8];
    add_scaled<T>(old, sum, P.scale, v);
    store_cols(row, col, P.dim, v);
}

// ---- gradient: few ids --------------------------------------------------------------------------------------------
// One launch.  A workgroup per position: it compares all ids with its own, leaves if one before it is the same, and else adds up
// the rows of those that are -- with few of them every wave has columns of its own, with many every wave has a quarter of the
// positions and the waves' sums are added in order.
constexpr int kDirectMany = 8, kDirectWords = (int)(kDirectIds / 64);

template <class G>
__device__ __forceinline__ void add_named(const G* __restrict__ grad, uint64_t stride, uint32_t col, uint32_t dim, const u64* words, int first, int step,
                                          float* sum) {
    for (int x = first; x < kDirectWords; x += step) {
        u64 m = words[x];
        m = (u64)(uint32_t)__builtin_amdgcn_readfirstlane((int)(m >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)m);   // the wave's own
        while (m) {
            float g[4][8];
            bool on[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                on[j] = m != 0;
                if (on[j]) {
                    const uint32_t pos = (uint32_t)x * 64 + (uint32_t)__builtin_ctzll(m);
                    m &= m - 1;
                    load_cols(grad + (uint64_t)pos * stride, col, dim, g[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (on[j]) {
#pragma unroll
                    for (int i = 0; i < 8; i++) sum[i] += g[j][i];
                }
            }
        }
    }
}

template <class G, class T>
__global__ __launch_bounds__(kGradThreads) void grad_direct_kernel(const int32_t* __restrict__ ids, uint32_t n, const uint64_t* n_dev, uint32_t rows,
                                                                   const G* __restrict__ grad, uint64_t grad_stride, uint32_t dim,
                                                                   T* __restrict__ table, uint64_t table_stride, float scale, int accumulate) {
    __shared__ u64 words[kDirectWords];
    __shared__ float acc[kGradThreads / 64 - 1][64][8];
    const uint32_t valid = (uint32_t)ids_that_count(n, n_dev);
    const int w = wave_id(), lane = lane_id();
    if (blockIdx.x >= n) {   // rows that no id names, when the gradient is written whole
        const uint64_t r0 = (uint64_t)(blockIdx.x - n) * kZeroRows;
        if (threadIdx.x == 0) words[0] = 0;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < valid; j += kGradThreads) {
            const uint64_t d = (uint64_t)(int64_t)ids[j] - r0;   // (below kZeroRows for these rows only)
            if (d < kZeroRows) atomicOr(&words[0], 1ull << d);
        }
        __syncthreads();
        zero_rows(table, table_stride, rows, dim, r0, words[0]);
        return;
    }
    const uint32_t t = blockIdx.x;
    if (t >= valid) return;
    const int32_t id = ids[t];
    if (id < 0 || (uint32_t)id >= rows) return;
    bool earlier = false;
    int many = 0;
#pragma unroll
    for (int x0 = 0; x0 < kDirectWords; x0 += kGradThreads / 64) {
        const int x = x0 + w;
        const uint32_t j = (uint32_t)x * 64 + lane;
        const u64 m = __ballot(j < valid && ids[j] == id);
        if (lane == 0) words[x] = m;
        if (m && (uint32_t)x * 64 + (uint32_t)__builtin_ctzll(m) < t) earlier = true;
        many += __popcll(m);
    }
    if (__syncthreads_or(earlier)) return;
    if (!__syncthreads_or(many > kDirectMany)) {   // (of one wave's words: at most four times as many in all)
        for (uint32_t col = (uint32_t)threadIdx.x * 8; col < dim; col += kGradThreads * 8) {
            float sum[8], old[8], v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] = old[i] = 0.f;
            T* row = table + (uint64_t)(uint32_t)id * table_stride;
            if (accumulate) load_cols(row, col, dim, old);
            add_named(grad, grad_stride, col, dim, words, 0, 1, sum);
            add_scaled<T>(old, sum, scale, v);
            store_cols(row, col, dim, v);
        }
        return;
    }
    for (uint32_t c0 = 0; c0 < dim; c0 += 512) {
        const uint32_t col = c0 + (uint32_t)lane * 8;
        const bool in = col < dim;
        float sum[8], old[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] = old[i] = 0.f;
        T* row = table + (uint64_t)(uint32_t)id * table_stride;
        if (in && w == 0 && accumulate) load_cols(row, col, dim, old);
        if (in) add_named(grad, grad_stride, col, dim, words, w, kGradThreads / 64, sum);
        if (w) {
#pragma unroll
            for (int i = 0; i < 8; i++) acc[w - 1][lane][i] = sum[i];
        }
        __syncthreads();
        if (w == 0 && in) {
            for (int x = 0; x < kGradThreads / 64 - 1; x++) {
#pragma unroll
                for (int i = 0; i < 8; i++) sum[i] += acc[x][lane][i];
            }
            add_scaled<T>(old, sum, scale, v);
            store_cols(row, col, dim, v);
        }
        __syncthreads();
    }
}

}  // namespace

hipError_t launch_embed(const EmbedArgs& A, hipStream_t stream) {
    if (A.n == 0) return hipSuccess;
    const uint64_t blocks = capped((A.n * ((A.dim + 7) / 8) + kEmbedTile - 1) / kEmbedTile);
    return with_dtype(A.dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_dtype(A.out_dtype, [&](auto o) {
            typedef decltype(o) O;
            return launch(embed_kernel<T, O>, blocks, kEmbedThreads, stream, A.ids, A.n, A.n_dev, (const T*)A.table, (uint32_t)A.rows, (uint32_t)A.dim, A.stride,
                          (O*)A.out, A.out_stride, A.scale);
        });
    });
}

hipError_t launch_embed_grad(const EmbedGradArgs& A, hipStream_t stream) {
    const uint32_t rows = (uint32_t)A.rows, dim = (uint32_t)A.dim;
    const uint64_t zero_blocks = A.accumulate ? 0 : (A.rows + kZeroRows - 1) / kZeroRows;
    if (A.n <= kDirectIds) {
        if (A.n + zero_blocks == 0) return hipSuccess;
        return with_dtype(A.table_dtype, [&](auto t) {
            typedef decltype(t) T;
            return with_dtype(A.dtype, [&](auto g) {
                typedef decltype(g) G;
                return launch(grad_direct_kernel<G, T>, A.n + zero_blocks, kGradThreads, stream, A.ids, (uint32_t)A.n, A.n_dev, rows, (const G*)A.grad, A.grad_stride, dim,
                              (T*)A.table, A.table_stride, A.scale, A.accumulate);
            });
        });
    }
    const GradWork W = grad_work(A.n, A.dim);
    uint8_t* base = (uint8_t*)A.work;
    uint32_t* const kb[2] = {(uint32_t*)(base + W.keys0), (uint32_t*)(base + W.keys1)};
    uint32_t* const pb[2] = {(uint32_t*)(base + W.pos0), (uint32_t*)(base + W.pos1)};
    uint32_t* hist = (uint32_t*)(base + W.hist);
    int bits = 1;
    while (bits < 32 && (rows >> bits)) bits++;            // keys are 0 .. rows
    const int passes = (bits + kSortBits - 1) / kSortBits, per = (bits + passes - 1) / passes;
    const uint64_t tiles = (A.n + kSortTile - 1) / kSortTile;
    const uint32_t mask = (1u << per) - 1;
    for (int p = 0; p < passes; p++) {
        const int shift = p * per, from = (p + 1) & 1, to = p & 1;
        const uint32_t *k = kb[from], *q = pb[from], *h = hist;
        hipError_t e = launch(p ? sort_count_kernel<false> : sort_count_kernel<true>, tiles, kSortThreads, stream, A.ids, k, A.n, A.n_dev, rows, shift, mask, hist);
        if (e != hipSuccess) return e;
        e = launch(p ? sort_place_kernel<false> : sort_place_kernel<true>, tiles, kSortThreads, stream, A.ids, k, q, A.n, A.n_dev, rows, shift, mask, per, h, kb[to], pb[to]);
        if (e != hipSuccess) return e;
    }
    const int to = (passes - 1) & 1;
    const uint32_t lanes = grad_lanes(A.dim), walkers = kGradThreads / lanes, col_tiles = (uint32_t)(((A.dim + 7) / 8 + lanes - 1) / lanes);
    const uint64_t walk_blocks = (W.chunks + walkers - 1) / walkers * col_tiles;
    GradWalk P{kb[to], pb[to], A.n, rows, W.chunk, W.chunks, lanes, col_tiles, walk_blocks, A.grad, A.grad_stride, dim, A.table, A.table_stride, A.scale,
               A.accumulate, (float*)(base + W.part), W.dim8};
    const uint32_t join_tiles = (uint32_t)((A.dim + 511) / 512);
    return with_dtype(A.table_dtype, [&](auto t) {
        typedef decltype(t) T;
        hipError_t e = with_dtype(A.dtype, [&](auto g) {
            typedef decltype(g) G;
            return launch(grad_walk_kernel<G, T>, walk_blocks + zero_blocks, kGradThreads, stream, P);
        });
        if (e != hipSuccess) return e;
        return launch(grad_join_kernel<T>, W.chunks * join_tiles, kGradThreads, stream, P, join_tiles);
    });
}

}  // namespace l3
