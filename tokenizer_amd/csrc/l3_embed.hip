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

// ---- lookup -------------------------------------------------------------------------------------------------------
// One thread, eight neighbouring columns of one row.
constexpr int kEmbedThreads = 256;

template <class T, class O>
__global__ __launch_bounds__(kEmbedThreads) void embed_kernel(const int32_t* ids, uint64_t n, const uint64_t* n_dev, const T* table,
                                                              uint64_t rows, uint64_t dim, uint64_t stride, O* out, uint64_t out_stride,
                                                              float scale) {
    const uint64_t per_row = (dim + 7) / 8, total = ids_that_count(n, n_dev) * per_row;
    for (uint64_t g = (uint64_t)blockIdx.x * kEmbedThreads + threadIdx.x; g < total; g += (uint64_t)gridDim.x * kEmbedThreads) {
        const uint64_t t = g / per_row, col = (g - t * per_row) * 8;
        const int32_t id = ids[t];
        const bool there = id >= 0 && (uint64_t)id < rows;
        const T* src = table + (there ? (uint64_t)id : 0) * stride + col;
        O* dst = out + t * out_stride + col;
        if (col + 8 <= dim) {
            float v[8];
            load8(src, v);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = there ? v[i] * scale : 0.f;
            store8(dst, v);
        } else {
            for (uint64_t i = 0; col + i < dim; i++) dst[i] = (O)(there ? (float)src[i] * scale : 0.f);
        }
    }
}

// ---- gradient: ids sorted -----------------------------------------------------------------------------------------
// Stable counting sort of (id, position) by digits, the lowest first.  An id that is no row, and a position that does not
// count, has the key n_rows and ends up behind all others.  A tile of kSortTile ids per workgroup:
//   sort_count_kernel    how often each digit occurs in the tile
//   sort_place_kernel    adds up the counts of the tiles before it, ranks the tile's ids and writes them to their places
constexpr int kSortThreads = 256, kSortWaves = kSortThreads / 64, kSortRounds = kSortTile / kSortThreads;

__device__ __forceinline__ uint32_t sort_key(const int32_t* ids, uint64_t i, uint64_t valid, uint32_t rows) {
    if (i >= valid) return rows;
    const int32_t id = ids[i];
    return id < 0 || (uint32_t)id >= rows ? rows : (uint32_t)id;
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const int32_t* ids, const uint32_t* keys, uint64_t n, const uint64_t* n_dev,
                                                                  uint32_t rows, int shift, uint32_t mask, uint32_t* hist) {
    __shared__ uint32_t cnt[kSortBins];
    for (int d = threadIdx.x; d < kSortBins; d += kSortThreads) cnt[d] = 0;
    __syncthreads();
    const uint64_t valid = FIRST ? ids_that_count(n, n_dev) : n, lo = (uint64_t)blockIdx.x * kSortTile;
#pragma unroll 4
    for (int k = 0; k < kSortRounds; k++) {
        const uint64_t i = lo + (uint64_t)k * kSortThreads + threadIdx.x;
        if (i < n) atomicAdd(&cnt[((FIRST ? sort_key(ids, i, valid, rows) : keys[i]) >> shift) & mask], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kSortBins; d += kSortThreads) hist[(uint64_t)blockIdx.x * kSortBins + d] = cnt[d];
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const int32_t* ids, const uint32_t* keys, const uint32_t* poss, uint64_t n,
                                                                  const uint64_t* n_dev, uint32_t rows, int shift, uint32_t mask, int bits,
                                                                  const uint32_t* hist, uint32_t* keys_out, uint32_t* pos_out) {
    __shared__ uint32_t cnt[kSortWaves][kSortBins];
    __shared__ uint32_t tmp[kSortWaves];
    const int tid = threadIdx.x, w = wave_id(), lane = lane_id();
    for (int d = tid; d < kSortWaves * kSortBins; d += kSortThreads) (&cnt[0][0])[d] = 0;
    // where the tile's ids of digit d start: all ids of smaller digits, then those of digit d in the tiles before
    constexpr int kPer = kSortBins / kSortThreads;
    uint32_t all[kPer], before[kPer];
#pragma unroll
    for (int k = 0; k < kPer; k++) all[k] = before[k] = 0;
    for (uint32_t b = 0; b < gridDim.x; b++) {
#pragma unroll
        for (int k = 0; k < kPer; k++) {
            const uint32_t c = hist[(uint64_t)b * kSortBins + tid * kPer + k];
            all[k] += c;
            if (b < blockIdx.x) before[k] += c;
        }
    }
    uint32_t sum = 0, total;
#pragma unroll
    for (int k = 0; k < kPer; k++) sum += all[k];
    uint32_t start = block_escan<kSortWaves>(sum, tmp, &total);   // (barriers inside: cnt is zero behind them)
#pragma unroll
    for (int k = 0; k < kPer; k++) { const uint32_t a = all[k]; all[k] = start + before[k]; start += a; }
    // ranks: a wave has kSortTile / kSortWaves ids in a row, 64 at a time
    const uint64_t valid = FIRST ? ids_that_count(n, n_dev) : n;
    const uint64_t lo = (uint64_t)blockIdx.x * kSortTile + (uint64_t)w * (kSortTile / kSortWaves);
    uint32_t key[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int k = 0; k < kSortRounds; k++) {
        const uint64_t i = lo + (uint64_t)k * 64 + lane;
        key[k] = i < n ? (FIRST ? sort_key(ids, i, valid, rows) : keys[i]) : 0;
    }
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
#pragma unroll
    for (int k = 0; k < kPer; k++) {
        uint32_t run = all[k];
        for (int v = 0; v < kSortWaves; v++) { const uint32_t c = cnt[v][tid * kPer + k]; cnt[v][tid * kPer + k] = run; run += c; }
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
// A walker goes through `chunk` sorted positions for eight columns a thread, in order.  A run of one id that lies inside the
// chunk is stored at once.  A run that crosses a border leaves its part in the workspace: part[2 c] of the run that came in
// from the chunk before, part[2 c + 1] of the run that starts here and goes on; grad_join_kernel adds these up in order, at the
// chunk where the run starts.  Nothing is added by atomics: the same ids give the same bits.
constexpr int kGradThreads = 256;

// lanes of a row, a power of two, and how many tiles of columns there are
inline uint32_t grad_lanes(uint64_t dim) {
    const uint64_t v = (dim + 7) / 8;
    uint32_t l = 1;
    while (l < v && l < (uint32_t)kGradThreads) l *= 2;
    return l;
}

template <class T>
__device__ __forceinline__ void load_cols(const T* p, uint64_t col, uint64_t dim, float* v) {
    if (col + 8 <= dim) { load8(p + col, v); return; }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = col + i < dim ? (float)p[col + i] : 0.f;
}
template <class T>
__device__ __forceinline__ void store_cols(T* p, uint64_t col, uint64_t dim, const float* v) {
    if (col + 8 <= dim) { store8(p + col, v); return; }
    for (int i = 0; i < 8; i++) if (col + i < dim) p[col + i] = (T)v[i];
}
template <class T>
__device__ __forceinline__ void put_row(T* row, uint64_t col, uint64_t dim, const float* sum, float scale, int accumulate) {
    float v[8];
    if (accumulate) {
        load_cols(row, col, dim, v);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += scale * sum[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = scale * sum[i];
    }
    store_cols(row, col, dim, v);
}

template <class G, class T>
__global__ __launch_bounds__(kGradThreads) void grad_walk_kernel(const uint32_t* keys, const uint32_t* poss, uint64_t n, uint32_t rows,
                                                                 uint32_t chunk, uint64_t chunks, uint32_t lanes, uint64_t col_tiles,
                                                                 const G* grad, uint64_t grad_stride, uint64_t dim, T* table,
                                                                 uint64_t table_stride, float scale, int accumulate, float* part,
                                                                 uint64_t dim8) {
    const uint32_t walkers = kGradThreads / lanes, me = threadIdx.x / lanes;
    const uint64_t groups = (chunks + walkers - 1) / walkers * col_tiles;
    for (uint64_t g = blockIdx.x; g < groups; g += gridDim.x) {
        const uint64_t c = g / col_tiles * walkers + me, col = ((g % col_tiles) * lanes + threadIdx.x % lanes) * 8;
        if (c >= chunks || col >= dim) continue;
        const uint64_t lo = c * chunk, hi = lo + chunk < n ? lo + chunk : n;
        uint32_t cur = keys[lo];
        if (cur >= rows) continue;
        bool came_in = lo > 0 && keys[lo - 1] == cur;
        float sum[8];
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] = 0.f;
        for (uint64_t i = lo; i < hi; i++) {
            const uint32_t k = keys[i];
            if (k != cur) {
                if (came_in) store8(part + (2 * c) * dim8 + col, sum);
                else put_row(table + (uint64_t)cur * table_stride, col, dim, sum, scale, accumulate);
                came_in = false;
                cur = k;
                if (k >= rows) break;
#pragma unroll
                for (int j = 0; j < 8; j++) sum[j] = 0.f;
            }
            float v[8];
            load_cols(grad + (uint64_t)poss[i] * grad_stride, col, dim, v);
#pragma unroll
            for (int j = 0; j < 8; j++) sum[j] += v[j];
        }
        if (cur >= rows) continue;
        const bool goes_on = hi < n && keys[hi] == cur;
        if (came_in) store8(part + (2 * c) * dim8 + col, sum);
        else if (goes_on) store8(part + (2 * c + 1) * dim8 + col, sum);
        else put_row(table + (uint64_t)cur * table_stride, col, dim, sum, scale, accumulate);
    }
}

template <class T>
__global__ __launch_bounds__(kGradThreads) void grad_join_kernel(const uint32_t* keys, uint64_t n, uint32_t rows, uint32_t chunk,
                                                                 uint64_t chunks, uint32_t lanes, uint64_t col_tiles, uint64_t dim,
                                                                 T* table, uint64_t table_stride, float scale, int accumulate,
                                                                 const float* part, uint64_t dim8) {
    const uint32_t walkers = kGradThreads / lanes, me = threadIdx.x / lanes;
    const uint64_t groups = (chunks + walkers - 1) / walkers * col_tiles;
    for (uint64_t g = blockIdx.x; g < groups; g += gridDim.x) {
        const uint64_t c = g / col_tiles * walkers + me, col = ((g % col_tiles) * lanes + threadIdx.x % lanes) * 8;
        const uint64_t lo = c * chunk, hi = lo + chunk;
        if (c >= chunks || col >= dim || hi >= n) continue;
        const uint32_t k = keys[hi - 1];
        if (k >= rows || keys[hi] != k || (lo > 0 && keys[lo - 1] == k)) continue;
        float sum[8], v[8];
        load8(part + (2 * c + 1) * dim8 + col, sum);
        for (uint64_t d = c + 1; d < chunks && keys[d * chunk] == k; d++) {
            load8(part + (2 * d) * dim8 + col, v);
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] += v[i];
        }
        put_row(table + (uint64_t)k * table_stride, col, dim, sum, scale, accumulate);
    }
}

// Rows that no id names, when the gradient is written whole.  A wave per row.
template <class T>
__global__ __launch_bounds__(kGradThreads) void grad_zero_kernel(const uint32_t* keys, uint64_t n, uint64_t rows, uint64_t dim, T* table,
                                                                 uint64_t table_stride) {
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (uint64_t r = (uint64_t)blockIdx.x * (kGradThreads / 64) + wave_id(); r < rows; r += (uint64_t)gridDim.x * (kGradThreads / 64)) {
        uint64_t a = 0, b = n;
        while (a < b) { const uint64_t m = (a + b) / 2; if (keys[m] < r) a = m + 1; else b = m; }
        if (a < n && keys[a] == r) continue;
        for (uint64_t col = (uint64_t)lane_id() * 8; col < dim; col += 512) store_cols(table + r * table_stride, col, dim, zero);
    }
}

}  // namespace

hipError_t launch_embed(const EmbedArgs& A, hipStream_t stream) {
    if (A.n == 0) return hipSuccess;
    const uint64_t blocks = capped((A.n * ((A.dim + 7) / 8) + kEmbedThreads - 1) / kEmbedThreads);
    return with_dtype(A.dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_dtype(A.out_dtype, [&](auto o) {
            typedef decltype(o) O;
            return launch(embed_kernel<T, O>, blocks, kEmbedThreads, stream, A.ids, A.n, A.n_dev, (const T*)A.table, A.rows, A.dim, A.stride,
                          (O*)A.out, A.out_stride, A.scale);
        });
    });
}

hipError_t launch_embed_grad(const EmbedGradArgs& A, hipStream_t stream) {
    const uint32_t rows = (uint32_t)A.rows;
    const GradWork W = grad_work(A.n, A.dim);
    uint8_t* base = (uint8_t*)A.work;
    uint32_t* keys = nullptr;
    uint32_t* poss = nullptr;
    if (A.n) {
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
            hipError_t e = p == 0 ? launch(sort_count_kernel<true>, tiles, kSortThreads, stream, A.ids, (const uint32_t*)kb[from], A.n, A.n_dev, rows, shift, mask, hist)
                                  : launch(sort_count_kernel<false>, tiles, kSortThreads, stream, A.ids, (const uint32_t*)kb[from], A.n, A.n_dev, rows, shift, mask, hist);
            if (e != hipSuccess) return e;
            e = p == 0 ? launch(sort_place_kernel<true>, tiles, kSortThreads, stream, A.ids, (const uint32_t*)kb[from], (const uint32_t*)pb[from], A.n, A.n_dev, rows, shift, mask, per, (const uint32_t*)hist, kb[to], pb[to])
                       : launch(sort_place_kernel<false>, tiles, kSortThreads, stream, A.ids, (const uint32_t*)kb[from], (const uint32_t*)pb[from], A.n, A.n_dev, rows, shift, mask, per, (const uint32_t*)hist, kb[to], pb[to]);
            if (e != hipSuccess) return e;
            keys = kb[to];
            poss = pb[to];
        }
    }
    const uint32_t lanes = grad_lanes(A.dim);
    const uint64_t col_tiles = ((A.dim + 7) / 8 + lanes - 1) / lanes, walkers = kGradThreads / lanes;
    const uint64_t blocks = capped((W.chunks + walkers - 1) / walkers * col_tiles);
    float* part = (float*)(base + W.part);
    return with_dtype(A.table_dtype, [&](auto t) {
        typedef decltype(t) T;
        hipError_t e = hipSuccess;
        if (!A.accumulate) {
            e = launch(grad_zero_kernel<T>, capped((A.rows + kGradThreads / 64 - 1) / (kGradThreads / 64)), kGradThreads, stream, (const uint32_t*)keys, A.n, A.rows, A.dim,
                       (T*)A.table, A.table_stride);
            if (e != hipSuccess) return e;
        }
        if (A.n == 0) return e;
        e = with_dtype(A.dtype, [&](auto g) {
            typedef decltype(g) G;
            return launch(grad_walk_kernel<G, T>, blocks, kGradThreads, stream, (const uint32_t*)keys, (const uint32_t*)poss, A.n, rows, W.chunk, W.chunks, lanes, col_tiles,
                          (const G*)A.grad, A.grad_stride, A.dim, (T*)A.table, A.table_stride, A.scale, A.accumulate, part, W.dim8);
        });
        if (e != hipSuccess) return e;
        return launch(grad_join_kernel<T>, blocks, kGradThreads, stream, (const uint32_t*)keys, A.n, rows, W.chunk, W.chunks, lanes, col_tiles, A.dim, (T*)A.table,
                      A.table_stride, A.scale, A.accumulate, (const float*)part, W.dim8);
    });
}

}  // namespace l3
