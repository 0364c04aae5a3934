// l3_embed.hip -- embedding lookup and its gradient.
//
//   out[t]  = scale * table[ids[t]]                       (an id outside [0, n_rows): a row of zeros)
//   table[v] (+)= scale * sum over {t : ids[t] = v} of grad[t]
//
// Products and sums are in 32 bits, rounded once where they are stored.
#include "l3_token_kernels.h"

#include <type_traits>

#include "l3_dev.h"

namespace l3 {

namespace {

__device__ __forceinline__ uint64_t ids_that_count(uint64_t n, const uint64_t* n_dev) {
    if (!n_dev) return n;
    const uint64_t m = *n_dev;
    return m < n ? m : n;
}

// A row is worked on in vectors of N columns.  The last of a row whose width is no multiple of N begins `skip` columns early, so that
// every load has N elements; those columns belong to the vector before.  Rows of fewer than eight columns (SMALL) are loaded one
// element at a time.
struct Cols { uint32_t col, skip; };
template <uint32_t N = 8>
__device__ __forceinline__ Cols cols_of(uint32_t vec, uint32_t dim) {
    const uint32_t c = vec * N;
    if (c + N <= dim || dim < 8) return {c, 0};
    return {dim - N, c + N - dim};
}
template <bool SMALL, bool ONCE = false, int N = 8, class T>
__device__ __forceinline__ typename Few<T, N>::V load_cols(const T* row, Cols c, uint32_t dim) {
    if constexpr (SMALL) {
        typename Few<T, N>::V v = (T)0.f;
        for (uint32_t i = 0; i < N; i++) if (c.col + i < dim) v[i] = row[c.col + i];
        return v;
    } else {
        return ONCE ? load8_once<N>(row + c.col) : load8<N>(row + c.col);
    }
}
// The vector's own columns; SHARED: the skipped ones hold the same values as their owner stores.
template <bool SMALL, bool SHARED, bool ONCE = false, int N = 8, class T>
__device__ __forceinline__ void store_cols(T* row, Cols c, uint32_t dim, typename Few<T, N>::F v) {
    if constexpr (SMALL) {
        for (uint32_t i = 0; i < N; i++) if (c.col + i < dim) row[c.col + i] = (T)v[i];
    } else if (SHARED || c.skip == 0) {
        ONCE ? store8_once<N>(row + c.col, v) : store8<N>(row + c.col, v);
    } else {
#pragma unroll
        for (uint32_t i = 1; i < N; i++) if (i >= c.skip) row[c.col + i] = (T)v[i];
    }
}

// ---- lookup -------------------------------------------------------------------------------------------------------
// A thread has PER times as many neighbouring columns as make 16 bytes of the output, all loads in flight before the first store.
// What is divided is a workgroup's first vector (once) and 32-bit offsets from it.  Bound by memory: 16,384 rows of 4,096 in 16 bits
// take 35.7 us with inputs in turn (56 MB of distinct rows read and 134 MB written: 5.3 TB/s, and 29 us at the rates of reading alone, 5.7,
// and of filling alone, 6.85), and 31 on the same inputs again, whose rows the last cache still has; 64 rows a launch (2.5 us).
//
// Outputs of 16 MiB and more (kEmbedOnce) pass the caches: stored the usual way, the output drives the table's rows out of them
// (the same inputs again: 44 us instead of 32 at the size above; 16,384 rows of 2,048 in 32 bits 46 and 32).  A smaller output stays in them for the
// kernel that reads it next.  One vector a thread is best up to 2^24 vectors (16,384 x 4,096: 32 us, with four 35), four above
// (65,536 x 4,096: 169 and 144).
constexpr int kEmbedThreads = 256;
constexpr uint64_t kEmbedOnce = 1u << 20, kEmbedMany = 1u << 24;   // vectors of 16 bytes

template <class T, class O, int PER, bool ONCE, bool SMALL>
__global__ __launch_bounds__(kEmbedThreads) void embed_kernel(const int32_t* __restrict__ ids, uint64_t n, const uint64_t* __restrict__ n_dev,
                                                              const T* __restrict__ table, uint32_t rows, uint32_t dim, uint64_t stride,
                                                              O* __restrict__ out, uint64_t out_stride, float scale) {
    constexpr uint32_t kTile = kEmbedThreads * PER;
    constexpr int N = 16 / sizeof(O);
    typedef typename Few<T, N>::F F;
    const uint32_t per_row = (dim + N - 1) / N;
    const uint64_t count = ids_that_count(n, n_dev), total = count * per_row;
    for (uint64_t g0 = (uint64_t)blockIdx.x * kTile; g0 < total; g0 += (uint64_t)gridDim.x * kTile) {
        const uint64_t t0 = g0 / per_row;
        const uint32_t r0 = (uint32_t)(g0 - t0 * per_row);
        uint64_t t[PER];
        Cols c[PER];
        int32_t id[PER];
        typename Few<T, N>::V v[PER];
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const uint32_t at = r0 + k * kEmbedThreads + threadIdx.x, row = at / per_row;
            t[k] = t0 + row;
            c[k] = cols_of<N>(at - row * per_row, dim);
            id[k] = ids[t[k] < count ? t[k] : count - 1];
        }
#pragma unroll
        for (int k = 0; k < PER; k++)   // (an id that is no row loads row 0 and stores zeros)
            v[k] = load_cols<SMALL, false, N>(table + (uint64_t)((uint32_t)id[k] < rows ? (uint32_t)id[k] : 0u) * stride, c[k], dim);
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const F x = __builtin_convertvector(v[k], F) * scale;
            if (t[k] < count) store_cols<SMALL, true, ONCE, N>(out + t[k] * out_stride, c[k], dim, (uint32_t)id[k] < rows ? x : (F)0.f);
        }
    }
}

// ---- gradient: ids sorted -----------------------------------------------------------------------------------------
// Stable counting sort of (id, position) by digits, the lowest first.  An id that is no row, and a position that does not
// count, has the key n_rows and ends up behind all others.  A tile of ids per workgroup:
//   sort_count_kernel    how often each digit occurs in the tile
//   sort_place_kernel    adds up the counts of the tiles before it, ranks the tile's ids and writes them to their places
// Bound by latency: 4.9 and 7.9 us a pass for 65,536 ids, two passes for up to 2^18 - 1 rows.  (Adding the counts up in every workgroup
// saves a launch for their scan; a look-back from tile to tile would need cleared flags.)
constexpr int kSortWaves = kSortThreads / 64;
static_assert(kSortThreads == 2 * kSortBins, "two threads a digit add up the tiles' counts");

__device__ __forceinline__ uint32_t sort_key(const int32_t* ids, uint64_t i, uint64_t valid, uint32_t rows) {
    if (i >= valid) return rows;
    const int32_t id = ids[i];
    return id < 0 || (uint32_t)id >= rows ? rows : (uint32_t)id;
}

template <bool FIRST, int ROUNDS>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const int32_t* ids, const uint32_t* keys, uint64_t n, const uint64_t* n_dev,
                                                                  uint32_t rows, int shift, uint32_t mask, uint32_t* hist) {
    __shared__ uint32_t cnt[kSortBins];
    if (threadIdx.x < kSortBins) cnt[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t valid = FIRST ? ids_that_count(n, n_dev) : n, lo = (uint64_t)blockIdx.x * kSortThreads * ROUNDS;
#pragma unroll
    for (int k = 0; k < ROUNDS; k++) {
        const uint64_t i = lo + (uint64_t)k * kSortThreads + threadIdx.x;
        if (i < n) atomicAdd(&cnt[((FIRST ? sort_key(ids, i, valid, rows) : keys[i]) >> shift) & mask], 1u);
    }
    __syncthreads();
    if (threadIdx.x < kSortBins) hist[(uint64_t)blockIdx.x * kSortBins + threadIdx.x] = cnt[threadIdx.x];
}

template <bool FIRST, int ROUNDS>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const int32_t* ids, const uint32_t* keys, const uint32_t* poss, uint64_t n,
                                                                  const uint64_t* n_dev, uint32_t rows, int shift, uint32_t mask, int bits,
                                                                  const uint32_t* hist, uint32_t* keys_out, uint32_t* pos_out) {
    __shared__ uint32_t cnt[kSortWaves][kSortBins];
    __shared__ uint32_t half_all[kSortBins], half_before[kSortBins];
    __shared__ uint32_t tmp[kSortWaves];
    const int tid = threadIdx.x, w = wave_id(), lane = lane_id();
    const uint64_t valid = FIRST ? ids_that_count(n, n_dev) : n;
    const uint64_t lo = ((uint64_t)blockIdx.x * kSortThreads + (uint64_t)w * 64) * ROUNDS;
    uint32_t key[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int k = 0; k < ROUNDS; k++) {
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
    // ranks: a wave has 64 ROUNDS ids in a row, 64 at a time
#pragma unroll
    for (int k = 0; k < ROUNDS; k++) {
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
    for (int k = 0; k < ROUNDS; k++) {
        const uint64_t i = lo + (uint64_t)k * 64 + lane;
        const uint32_t at = cnt[w][(key[k] >> shift) & mask] + rank[k];
        if (i < n && at < n) {   // (always, unless the ids or the workspace change under the call)
            keys_out[at] = key[k];
            pos_out[at] = FIRST ? (uint32_t)i : poss[i];
        }
    }
}

// ---- gradient: ids ranked -----------------------------------------------------------------------------------------
// Up to kRankIds ids in one launch: the place of position i is the number of positions j with key_j < key_i, or key_j = key_i and
// j < i.  A workgroup has kRankMine positions and all keys in LDS; each of its 32 half waves counts over a part of them, four keys
// a load.  Bound by the n^2 comparisons: 7 us for 5,003 ids.  Whole gradients of 64 .. 256 columns, ranked / sorted by digits (us):
// 8,192 ids 20 / 28, 12,288 34 / 33, 16,384 40 / 33.
constexpr uint32_t kRankMine = 32;

__global__ __launch_bounds__(kSortThreads) void sort_rank_kernel(const int32_t* __restrict__ ids, uint32_t n, const uint64_t* __restrict__ n_dev, uint32_t rows,
                                                                 uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out) {
    __shared__ __align__(16) uint32_t key[kRankIds];
    __shared__ uint32_t rank[kRankMine];
    const uint32_t valid = (uint32_t)ids_that_count(n, n_dev), i0 = blockIdx.x * kRankMine;
    constexpr uint32_t kParts = kSortThreads / kRankMine;
    const uint32_t quads = (n + 4 * kParts - 1) / (4 * kParts), all = quads * 4 * kParts;   // (kRankIds is a multiple of 4 kParts)
    constexpr int kPer = (int)(kRankIds / kSortThreads);
    int32_t id[kPer];
#pragma unroll
    for (int x = 0; x < kPer; x++) {
        const uint32_t j = (uint32_t)x * kSortThreads + threadIdx.x;
        id[x] = j < valid ? ids[j] : -1;
    }
#pragma unroll
    for (int x = 0; x < kPer; x++) {
        const uint32_t j = (uint32_t)x * kSortThreads + threadIdx.x;
        if (j < all) key[j] = j >= n ? ~0u : id[x] < 0 || (uint32_t)id[x] >= rows ? rows : (uint32_t)id[x];
    }
    if (threadIdx.x < kRankMine) rank[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t i = i0 + threadIdx.x % kRankMine, part = threadIdx.x / kRankMine, k = key[i];   // (i < all: all is a multiple of kRankMine)
    uint32_t count = 0;
    const uint32_t lo = part * quads * 4;
#pragma unroll 4
    for (uint32_t q = 0; q < quads; q++) {
        const uint32_t j = lo + q * 4, bound = k + (j < i0 ? 1u : 0u);   // before the workgroup's own positions an equal key counts
        const uint4 v = *reinterpret_cast<const uint4*>(&key[j]);
        count += (v.x < bound) + (v.y < bound) + (v.z < bound) + (v.w < bound);
    }
    if (part == 0) for (uint32_t j = i0; j < i0 + kRankMine; j++) count += j < i && key[j] == k ? 1u : 0u;
    count += __shfl_xor(count, 32, 64);
    if (!(threadIdx.x & 32)) atomicAdd(&rank[threadIdx.x % kRankMine], count);
    __syncthreads();
    if (part == 0 && i < n) {
        keys_out[rank[threadIdx.x]] = k;
        pos_out[rank[threadIdx.x]] = i;
    }
}

// ---- gradient: runs of one id added up ----------------------------------------------------------------------------
// A wave walks through `chunk` sorted positions for 512 columns, in order, eight at a time: the eight rows of the gradient and, where
// a run of one id ends, the row of the table it is added to are loaded together.  Keys and positions of the whole chunk are in
// one register each (lane j has position j).  A run that lies inside the chunk is stored at once.  The parts of a run that crosses
// from one wave of a workgroup to the next meet in LDS; a run that crosses the workgroup's border leaves its part in the
// workspace: part[2 b] of the run that came in from the workgroup before, part[2 b + 1] of the run that starts here and goes
// on; grad_join_kernel adds these up at the workgroup where the run starts.  Nothing is added by atomics: the same ids give the
// same bits.  What comes from the workspace is held to the arrays' bounds, so that a workspace shared by mistake gives wrong sums and
// no access outside them.
//
// Bound by memory: 65,536 ids onto 32-bit gradients of 128,256 x 4,096 read 0.81 GB and write 0.32 GB (counters: the distinct rows,
// each once, and 4 % for the parts) in 250 us, 4.5 TB/s; a copy of 4 GiB reaches 4.7.  Rows in flight, us of the whole call: two 308,
// four 279, eight 265; loading the next eight while these are added up gains nothing more (268).  Keys and positions in
// registers instead of a load each, and no loads by element at the row's end: 346 -> 272 us.
constexpr int kGradThreads = 64 * kGradWaves;
constexpr int kGradGroup = 8;
constexpr uint32_t kGradCols = 512;
// A gradient above the last cache's 256 MiB is loaded past the caches (65,536 x 4,096 in 16 bits: 288 us instead of 313); a smaller one
// may still be in them from the kernel that made it (8,192 x 4,096: 55 instead of 48 us if it is loaded past them).
constexpr uint64_t kGradOnce = 256ull << 20;
// Rows a workgroup looks after when the gradient is written whole.  128,256 rows of 4,096 in 32 bits / of 64 in 16 bits, us: 8 rows
// 397 / 36, 16 rows 401 / 28, 32 rows 409 / 25, 64 rows 415 / 24.
constexpr uint32_t kZeroRows = 32;

// Rows [r0, r0 + kZeroRows) of which `named` has no mark become zero; by a whole workgroup.  16 bytes a lane, the last ones of a row
// overlapping those before.
template <bool SMALL, class T>
__device__ __forceinline__ void zero_rows(T* table, uint64_t table_stride, uint64_t rows, uint32_t dim, uint64_t r0, const uint32_t* named) {
    constexpr int N = 16 / sizeof(T);
    const uint32_t per_row = (dim + N - 1) / N;
    for (uint32_t j = wave_id(); j < kZeroRows && r0 + j < rows; j += kGradWaves) {
        if (named[j]) continue;
        for (uint32_t k = lane_id(); k < per_row; k += 64)
            store_cols<SMALL, true, false, N>(table + (r0 + j) * table_stride, cols_of<N>(k, dim), dim, (typename Few<T, N>::F)0.f);
    }
}

// The first position of the sorted keys that is not below r, 64 places at a time, by a whole wave.
__device__ __forceinline__ uint64_t first_key(const uint32_t* __restrict__ keys, uint64_t n, uint64_t r) {
    uint64_t lo = 0, len = n;                // the keys before lo are below r, key lo + len is not
    while (len) {
        const uint64_t step = (len + 63) / 64, at = lo + ((uint64_t)lane_id() + 1) * step - 1;
        const u64 below = __ballot(at < lo + len && keys[at < lo + len ? at : lo] < r);
        const uint64_t k = (uint64_t)__popcll(below);                     // (keys ascend: the low lanes)
        lo += k * step;
        len = len - k * step < step ? len - k * step : step - 1;
    }
    return lo;
}

struct GradWalk {
    uint64_t n; uint32_t rows;
    uint32_t chunk, tiles; uint64_t walk_blocks;
    uint64_t grad_stride; uint32_t dim;
    uint64_t table_stride;
    float scale; int accumulate;
    uint64_t dim8;
};

__device__ __forceinline__ uint32_t of_lane(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }

template <class G, class T, bool ONCE, bool SMALL>
__global__ __launch_bounds__(kGradThreads) void grad_walk_kernel(GradWalk P, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ poss,
                                                                 const G* __restrict__ grad, T* __restrict__ table, float* __restrict__ part) {
    const uint32_t rows = P.rows, dim = P.dim;
    if (blockIdx.x >= P.walk_blocks) {   // rows that no id names, when the gradient is written whole
        __shared__ uint32_t named[kZeroRows];
        __shared__ uint64_t ends[2];
        const uint64_t r0 = (uint64_t)(blockIdx.x - P.walk_blocks) * kZeroRows;
        if (threadIdx.x < kZeroRows) named[threadIdx.x] = 0;
        if (wave_id() < 2) ends[wave_id()] = first_key(keys, P.n, r0 + wave_id() * kZeroRows);
        __syncthreads();
        for (uint64_t i = ends[0] + threadIdx.x; i < ends[1]; i += kGradThreads) if (keys[i] - r0 < kZeroRows) named[keys[i] - r0] = 1;
        __syncthreads();
        zero_rows<SMALL>(table, P.table_stride, rows, dim, r0, named);
        return;
    }
    __shared__ F8 heads[kGradWaves][64];
    __shared__ bool goes_through[kGradWaves];
    const uint64_t block = blockIdx.x / P.tiles;
    const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane((int)wave_id());
    const uint64_t c = block * kGradWaves + w, lo = c * P.chunk < P.n ? c * P.chunk : P.n;
    const uint32_t vec = (uint32_t)(blockIdx.x - block * P.tiles) * 64 + lane_id(), len = lo + P.chunk < P.n ? P.chunk : (uint32_t)(P.n - lo);
    const uint32_t key = (uint32_t)lane_id() < len ? keys[lo + lane_id()] : ~0u, pos = (uint32_t)lane_id() < len ? min(poss[lo + lane_id()], (uint32_t)P.n - 1) : 0;
    // the key behind the chunk, and the run that came in, if one did
    const uint32_t behind = lo + len < P.n ? keys[lo + len] : ~0u, first = of_lane(key, 0), in_front = lo && len ? keys[lo - 1] : ~0u;
    const uint32_t came_in = first == in_front && first < rows ? first : ~0u;
    const u64 none = __ballot(key >= rows);                           // ids that are no rows come last
    const uint32_t used = none ? (uint32_t)__builtin_ctzll(none) : 64;
    const bool mine = vec * 8 < dim;
    const Cols at = cols_of(mine ? vec : 0, dim);
    F8 sum = 0.f, head = 0.f;
    for (uint32_t i = 0; i < used; i += kGradGroup) {
        uint32_t k[kGradGroup + 1];
        typename Eight<G>::V g[kGradGroup];
        typename Eight<T>::V old[kGradGroup];
#pragma unroll
        for (int j = 0; j <= kGradGroup; j++) k[j] = i + j < len ? of_lane(key, i + j) : behind;
#pragma unroll
        for (int j = 0; j < kGradGroup; j++) {
            const uint32_t x = i + j < used ? i + j : used - 1;
            g[j] = load_cols<SMALL, ONCE>(grad + (uint64_t)of_lane(pos, x) * P.grad_stride, at, dim);
        }
#pragma unroll
        for (int j = 0; j < kGradGroup; j++) {
            old[j] = (T)0.f;
            if (i + j < used && k[j + 1] != k[j] && k[j] != came_in && P.accumulate) old[j] = load_cols<SMALL>(table + (uint64_t)k[j] * P.table_stride, at, dim);
        }
#pragma unroll
        for (int j = 0; j < kGradGroup; j++) {
            if (i + j >= used) break;
            sum += to_f8(g[j]);
            if (k[j + 1] == k[j]) continue;
            if (k[j] == came_in) head = sum;
            else if (mine) store_cols<SMALL, false>(table + (uint64_t)k[j] * P.table_stride, at, dim, to_f8(old[j]) + sum * P.scale);
            sum = 0.f;
        }
    }
    const uint32_t last = len ? of_lane(key, (int)len - 1) : ~0u;
    const bool goes_on = last < rows && last == behind, through = goes_on && last == came_in, starts = goes_on && !through;
    if (through) head = sum;
    if (w && came_in != ~0u) {
        heads[w][lane_id()] = head;
        goes_through[w] = through;
    }
    __syncthreads();
    // the run that this wave has to look after: the one that starts here and goes on or, in the first wave, the one that came in
    F8 x = starts ? sum : head;
    uint32_t v = w;
    bool on = goes_on;
    if (starts || (w == 0 && came_in != ~0u)) {
        while (on && ++v < kGradWaves) {
            x += heads[v][lane_id()];
            on = goes_through[v];
        }
        if (mine) {
            if (!starts) {
                store8(part + (2 * block) * P.dim8 + vec * 8, x);
            } else if (on) {
                store8(part + (2 * block + 1) * P.dim8 + vec * 8, x);
            } else {
                typename Eight<T>::V old = (T)0.f;
                T* row = table + (uint64_t)last * P.table_stride;
                if (P.accumulate) old = load_cols<SMALL>(row, at, dim);
                store_cols<SMALL, false>(row, at, dim, to_f8(old) + x * P.scale);
            }
        }
    }
    // (the first wave may have both: a run that came in and ended, and one that starts and goes on)
    if (w == 0 && starts && came_in != ~0u && mine) store8(part + (2 * block) * P.dim8 + vec * 8, head);
}

// Parts of long runs: a workgroup per walking workgroup and 512 columns, every wave a share of the parts, eight loads in flight.  Most
// workgroups find no run to join and leave after one load; 65,536 ids of which 6 % are the same: 7.5 us (26 us with one wave for
// all parts of a run and parts of single waves).
constexpr int kJoinGroup = 8;

template <class T, bool SMALL>
__global__ __launch_bounds__(kGradThreads) void grad_join_kernel(GradWalk P, const uint32_t* __restrict__ keys, T* __restrict__ table,
                                                                 const float* __restrict__ part) {
    __shared__ F8 acc[kGradWaves - 1][64];
    const uint64_t b = blockIdx.x / P.tiles, span = (uint64_t)P.chunk * kGradWaves;
    const uint32_t vec = (blockIdx.x - (uint32_t)b * P.tiles) * 64 + lane_id();
    const uint64_t lo = b * span, hi = lo + span;
    if (hi >= P.n) return;
    const uint32_t k = keys[hi - 1], behind = keys[hi], in_front = lo ? keys[lo - 1] : ~0u;
    if (k >= P.rows || behind != k || in_front == k) return;
    uint64_t more = 0;   // workgroups behind b that the run comes into
    for (;;) {
        const uint64_t at = hi + (more + lane_id()) * span;
        const u64 m = __ballot(at < P.n && keys[at] == k);
        if (m == ~0ull) { more += 64; continue; }
        more += (uint64_t)__builtin_ctzll(~m);
        break;
    }
    const int w = __builtin_amdgcn_readfirstlane((int)wave_id());
    const bool mine = vec * 8 < P.dim;
    const Cols at = cols_of(mine ? vec : 0, P.dim);
    T* row = table + (uint64_t)k * P.table_stride;
    const float* from = part + (uint64_t)(mine ? vec : 0) * 8;
    typename Eight<T>::V old = (T)0.f;
    F8 sum = 0.f;
    if (w == 0) {
        if (P.accumulate) old = load_cols<SMALL>(row, at, P.dim);
        sum = load8(from + (2 * b + 1) * P.dim8);
    }
    const uint64_t end = b + 1 + more * (w + 1) / kGradWaves;
    for (uint64_t d = b + 1 + more * w / kGradWaves; d < end; d += kJoinGroup) {
        F8 v[kJoinGroup];
#pragma unroll
        for (int j = 0; j < kJoinGroup; j++) v[j] = load8(from + 2 * (d + j < end ? d + j : end - 1) * P.dim8);
#pragma unroll
        for (int j = 0; j < kJoinGroup; j++) if (d + j < end) sum += v[j];
    }
    if (w) acc[w - 1][lane_id()] = sum;
    __syncthreads();
    if (w || !mine) return;
    for (int x = 0; x < kGradWaves - 1; x++) sum += acc[x][lane_id()];
    store_cols<SMALL, false>(row, at, P.dim, to_f8(old) + sum * P.scale);
}

// ---- gradient: few ids --------------------------------------------------------------------------------------------
// One launch, nothing sorted.  A workgroup per position and 512 columns: it compares all ids with its own, leaves if one before it
// is the same, and else adds up the rows of those that are, every wave a quarter of them.  Its own row and the table's are on
// their way while it compares.  Bound by the chain ids -> rows -> store: 5.4 us for 512 ids of 2,048 columns, 5.0 a call among others
// (sorted: 16 us).  WORDS * 64 ids are compared whatever n is, so there is a kernel each for 512, 1,024 and 2,048 of them: 512 ids of
// 2,048 columns take 6.7 us in the one for 2,048.
constexpr int kDirectGroup = 8;

template <class G, class T, bool SMALL, int WORDS>
__global__ __launch_bounds__(kGradThreads) void grad_direct_kernel(const int32_t* __restrict__ ids, uint32_t n, const uint64_t* n_dev, uint32_t rows,
                                                                   const G* __restrict__ grad, uint64_t grad_stride, uint32_t dim,
                                                                   T* __restrict__ table, uint64_t table_stride, float scale, int accumulate,
                                                                   uint32_t tiles) {
    __shared__ u64 words[WORDS];
    __shared__ uint32_t list[WORDS * 64];
    __shared__ F8 acc[kGradWaves - 1][64];
    const uint32_t valid = (uint32_t)ids_that_count(n, n_dev);
    const int w = __builtin_amdgcn_readfirstlane((int)wave_id()), lane = lane_id();
    if (blockIdx.x >= n * tiles) {   // rows that no id names, when the gradient is written whole
        const uint64_t r0 = (uint64_t)(blockIdx.x - n * tiles) * kZeroRows;
        if (threadIdx.x < kZeroRows) list[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < valid; j += kGradThreads) {
            const uint64_t d = (uint64_t)(int64_t)ids[j] - r0;   // (below kZeroRows for these rows only)
            if (d < kZeroRows) list[d] = 1;
        }
        __syncthreads();
        zero_rows<SMALL>(table, table_stride, rows, dim, r0, list);
        return;
    }
    const uint32_t t = blockIdx.x / tiles;
    if (t >= valid) return;
    int32_t other[WORDS / kGradWaves];
#pragma unroll
    for (int y = 0; y < WORDS / kGradWaves; y++) {
        const uint32_t j = (uint32_t)(y * kGradWaves + w) * 64 + lane;
        other[y] = ids[j < valid ? j : 0];
    }
    const int32_t id = ids[t];
    if (id < 0 || (uint32_t)id >= rows) return;
    const uint32_t vec = (blockIdx.x - t * tiles) * 64 + lane;
    const bool mine = vec * 8 < dim;
    const Cols at = cols_of(mine ? vec : 0, dim);
    T* row = table + (uint64_t)(uint32_t)id * table_stride;
    typename Eight<T>::V old = (T)0.f;
    F8 sum = 0.f;
    if (w == 0) {
        if (accumulate) old = load_cols<SMALL>(row, at, dim);
        sum = to_f8(load_cols<SMALL>(grad + (uint64_t)t * grad_stride, at, dim));
    }
    bool earlier = false;
#pragma unroll
    for (int y = 0; y < WORDS / kGradWaves; y++) {
        const int x = y * kGradWaves + w;
        const uint32_t j = (uint32_t)x * 64 + lane;
        const u64 m = __ballot(j < valid && j != t && other[y] == id);
        if (lane == 0) words[x] = m;
        if (m && (uint32_t)x * 64 + (uint32_t)__builtin_ctzll(m) < t) earlier = true;
    }
    if (__syncthreads_or(earlier)) return;
    // the others, in order: every wave knows how many there are in the words before its own
    static_assert(WORDS <= 64, "a lane a word");
    const u64 mine_word = lane < WORDS ? words[lane] : 0;
    const uint32_t upto = wave_iscan((uint32_t)__popcll(mine_word)), count = of_lane(upto, 63);
    if (count) {
        for (int x = w; x < WORDS; x += kGradWaves) {
            const u64 m = words[x];
            if ((m >> lane) & 1) list[of_lane(upto, x) - (uint32_t)__popcll(m) + (uint32_t)__popcll(m & ((1ull << lane) - 1))] = (uint32_t)x * 64 + lane;
        }
        __syncthreads();
        const uint32_t hi = count * (w + 1) / kGradWaves;
        for (uint32_t i = count * w / kGradWaves; i < hi; i += kDirectGroup) {
            typename Eight<G>::V g[kDirectGroup];
#pragma unroll
            for (int j = 0; j < kDirectGroup; j++) {
                const uint32_t p = (uint32_t)__builtin_amdgcn_readfirstlane((int)list[i + j < hi ? i + j : hi - 1]);
                g[j] = load_cols<SMALL>(grad + (uint64_t)p * grad_stride, at, dim);
            }
#pragma unroll
            for (int j = 0; j < kDirectGroup; j++) if (i + j < hi) sum += to_f8(g[j]);
        }
        if (w) acc[w - 1][lane] = sum;
        __syncthreads();
    }
    if (w || !mine) return;
    if (count) for (int x = 0; x < kGradWaves - 1; x++) sum += acc[x][lane];
    store_cols<SMALL, false>(row, at, dim, to_f8(old) + sum * scale);
}

// f(std::true_type / false_type): rows of fewer than eight columns, or not
template <class F>
hipError_t with_small(uint64_t dim, F f) {
    return dim < 8 ? f(std::true_type()) : f(std::false_type());
}

}  // namespace

hipError_t launch_embed(const EmbedArgs& A, hipStream_t stream) {
    if (A.n == 0) return hipSuccess;
    const uint64_t per = 16 / dtype_size(A.out_dtype), vectors = A.n * ((A.dim + per - 1) / per);
    return with_dtype(A.dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_dtype(A.out_dtype, [&](auto o) {
            typedef decltype(o) O;
            return with_small(A.dim, [&](auto small) {
                const int many = vectors >= kEmbedMany ? 4 : 1;
                auto* kernel = vectors >= kEmbedMany   ? embed_kernel<T, O, 4, true, small.value>
                               : vectors >= kEmbedOnce ? embed_kernel<T, O, 1, true, small.value>
                                                       : embed_kernel<T, O, 1, false, small.value>;
                const uint64_t tile = (uint64_t)kEmbedThreads * many;
                return launch(kernel, capped((vectors + tile - 1) / tile), kEmbedThreads, stream, A.ids, A.n, A.n_dev, (const T*)A.table, (uint32_t)A.rows,
                              (uint32_t)A.dim, A.stride, (O*)A.out, A.out_stride, A.scale);
            });
        });
    });
}

hipError_t launch_embed_grad(const EmbedGradArgs& A, hipStream_t stream) {
    const uint32_t rows = (uint32_t)A.rows, dim = (uint32_t)A.dim;
    const uint64_t zero_blocks = A.accumulate ? 0 : (A.rows + kZeroRows - 1) / kZeroRows;
    auto with_types = [&](auto f) {
        return with_dtype(A.table_dtype, [&](auto t) {
            return with_dtype(A.dtype, [&](auto g) { return with_small(A.dim, [&](auto small) { return f(g, t, small); }); });
        });
    };
    const uint32_t col_tiles = (dim + kGradCols - 1) / kGradCols;
    if (grad_direct(A.n, A.dim)) {
        if (A.n + zero_blocks == 0) return hipSuccess;
        return with_types([&](auto g, auto t, auto small) {
            typedef decltype(g) G;
            typedef decltype(t) T;
            auto* kernel = A.n <= 512    ? grad_direct_kernel<G, T, small.value, 8>
                           : A.n <= 1024 ? grad_direct_kernel<G, T, small.value, 16>
                                         : grad_direct_kernel<G, T, small.value, (int)(kDirectIds / 64)>;
            return launch(kernel, A.n * col_tiles + zero_blocks, kGradThreads, stream, A.ids, (uint32_t)A.n, A.n_dev, rows, (const G*)A.grad, A.grad_stride, dim,
                          (T*)A.table, A.table_stride, A.scale, A.accumulate, col_tiles);
        });
    }
    const GradWork W = grad_work(A.n, A.dim);
    uint8_t* base = (uint8_t*)A.work;
    uint32_t* const kb[2] = {(uint32_t*)(base + W.keys0), (uint32_t*)(base + W.keys1)};
    uint32_t* const pb[2] = {(uint32_t*)(base + W.pos0), (uint32_t*)(base + W.pos1)};
    uint32_t* hist = (uint32_t*)(base + W.hist);
    const uint32_t *keys = kb[0], *poss = pb[0];
    if (A.n <= kRankIds) {
        const hipError_t e = launch(sort_rank_kernel, (A.n + kRankMine - 1) / kRankMine, kSortThreads, stream, A.ids, (uint32_t)A.n, A.n_dev, rows, kb[0], pb[0]);
        if (e != hipSuccess) return e;
    } else {
        int bits = 1;
        while (bits < 32 && (rows >> bits)) bits++;            // keys are 0 .. rows
        const int passes = (bits + kSortBits - 1) / kSortBits, per = (bits + passes - 1) / passes;
        const uint64_t tiles = sort_tiles(A.n);
        const uint32_t mask = (1u << per) - 1;
        auto pass = [&](auto first, auto rounds, int shift, const uint32_t* k, const uint32_t* q, uint32_t* k_out, uint32_t* q_out) {
            const hipError_t e = launch(sort_count_kernel<first.value, rounds.value>, tiles, kSortThreads, stream, A.ids, k, A.n, A.n_dev, rows, shift, mask, hist);
            if (e != hipSuccess) return e;
            return launch(sort_place_kernel<first.value, rounds.value>, tiles, kSortThreads, stream, A.ids, k, q, A.n, A.n_dev, rows, shift, mask, per,
                          (const uint32_t*)hist, k_out, q_out);
        };
        auto pass_of = [&](auto rounds, int p) {
            const int from = (p + 1) & 1, to = p & 1;
            return p ? pass(std::false_type(), rounds, p * per, kb[from], pb[from], kb[to], pb[to])
                     : pass(std::true_type(), rounds, 0, kb[from], pb[from], kb[to], pb[to]);
        };
        for (int p = 0; p < passes; p++) {
            const int r = sort_rounds(A.n);
            const hipError_t e = r == 1   ? pass_of(std::integral_constant<int, 1>(), p)
                                 : r == 2 ? pass_of(std::integral_constant<int, 2>(), p)
                                          : pass_of(std::integral_constant<int, 4>(), p);
            if (e != hipSuccess) return e;
            keys = kb[p & 1];
            poss = pb[p & 1];
        }
    }
    const uint64_t walk_blocks = W.blocks * col_tiles;
    const GradWalk P{A.n, rows, W.chunk, col_tiles, walk_blocks, A.grad_stride, dim, A.table_stride, A.scale, A.accumulate, W.dim8};
    float* part = (float*)(base + W.part);
    return with_types([&](auto g, auto t, auto small) {
        typedef decltype(g) G;
        typedef decltype(t) T;
        const bool once = A.n * A.dim * sizeof(G) > kGradOnce;
        hipError_t e = launch(once ? grad_walk_kernel<G, T, true, small.value> : grad_walk_kernel<G, T, false, small.value>, walk_blocks + zero_blocks, kGradThreads, stream, P, keys, poss, (const G*)A.grad, (T*)A.table, part);
        if (e != hipSuccess) return e;
        return launch(grad_join_kernel<T, small.value>, walk_blocks, kGradThreads, stream, P, keys, (T*)A.table, (const float*)part);
    });
}

}  // namespace l3
