// l3_verify.hip -- verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Request i has k drafted tokens d_0 .. d_{k-1}, drawn from the rows q_j, and the target's rows p_0 .. p_k.  Token j is accepted
// while u_j q_j(d_j) < p_j(d_j); the first that is not (or, if all are, position k) is drawn anew: the smallest v with
//     w(0) + .. + w(v) > r (w(0) + .. + w(vocab - 1)),   w = max(p_a - q_a, 0) if token a was rejected, p_k if all were accepted,
// so that what comes out is distributed as the target's own tokens.  Without q the drafted token counts as certain (q = 1 there).
// Products, differences and sums are in 64 bits: the answer is a whole number, and a border must not move with the order.
//
// Only the rows at position a are read whole, so what the verification cannot do without is one row of p and one of q a request.  Two
// launches: the sums of kVerifyChunk entries by all workgroups, then a workgroup per request for the place of the border -- a draw
// needs the sum of the whole row, and one workgroup would read a row of 128,256 at the rate of one CU.
#include "l3_token_kernels.h"

#include "l3_dev.h"

namespace l3 {

namespace {

constexpr int kVerifyThreads = 256;

using Verdict = VerifyVerdict;

// Called by a whole wave.
template <class T>
__device__ Verdict verdict_of(const VerifyArgs& A, uint64_t i) {
    Verdict R;
    R.state = kBadRequest; R.a = 0; R.p_row = R.q_row = 0; R.token = -1;
    const uint64_t lo = A.off[i], hi = A.off[i + 1];
    if (lo > hi || hi > A.n_draft || hi - lo > A.max_draft) return R;
    const uint32_t k = (uint32_t)(hi - lo);
    uint32_t a = k;
    for (uint32_t j0 = 0; j0 < k; j0 += 64) {
        const uint32_t j = j0 + lane_id();
        bool ok = true;
        if (j < k) {
            const int32_t d = A.draft[lo + j];
            ok = false;
            if (d >= 0 && (uint64_t)d < A.vocab) {
                const double p = (double)(float)((const T*)A.target)[(lo + i + j) * A.target_stride + (uint64_t)d];
                const double q = A.q ? (double)(float)((const T*)A.q)[(lo + j) * A.q_stride + (uint64_t)d] : 1.0;
                ok = (double)A.u_accept[lo + j] * q < p;
            }
        }
        const u64 no = __ballot(!ok);
        if (no) { a = j0 + (uint32_t)__builtin_ctzll(no); break; }
    }
    R.a = a;
    R.p_row = lo + i + a;
    R.q_row = lo + a;
    R.state = a == k ? kDrawTarget : kDrawRest;
    if (a < k) R.token = A.draft[lo + a];
    return R;
}

// A weight that is no positive finite number counts as none.
__device__ __forceinline__ double weight(double x) { return x > 0.0 && x < __builtin_huge_val() ? x : 0.0; }

// Eight neighbouring entries: rest = what is left of the target after the draft, full = the target's own.
template <class T>
__device__ __forceinline__ void weights8(const VerifyArgs& A, const Verdict& R, uint64_t col, double* rest, double* full) {
    const T* p = (const T*)A.target + R.p_row * A.target_stride;
    const T* q = R.state == kDrawRest && A.q ? (const T*)A.q + R.q_row * A.q_stride : nullptr;
    F8 pv = 0.f, qv = 0.f;
    if (col + 8 <= A.vocab) {
        pv = to_f8(load8(p + col));
        if (q) qv = to_f8(load8(q + col));
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const bool in = col + j < A.vocab;
            pv[j] = in ? (float)p[col + j] : 0.f;
            if (q) qv[j] = in ? (float)q[col + j] : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        full[j] = weight((double)pv[j]);
        rest[j] = q ? weight((double)pv[j] - (double)qv[j]) : (uint64_t)(int64_t)R.token == col + j ? 0.0 : full[j];
    }
}

// Inclusive sums over the wave's lanes, by DPP as wave_iscan (l3_dev.h) has them.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double dpp_move_f64(double v) {
    const u64 b = (u64)__double_as_longlong(v);
    return __longlong_as_double((long long)((u64)dpp_move<CTRL, ROWS>((uint32_t)(b >> 32)) << 32 | dpp_move<CTRL, ROWS>((uint32_t)b)));
}
__device__ __forceinline__ double wave_iscan_f64(double v) {
    v += dpp_move_f64<0x111>(v);
    v += dpp_move_f64<0x112>(v);
    v += dpp_move_f64<0x114>(v);
    v += dpp_move_f64<0x118>(v);
    v += dpp_move_f64<0x142, 0xA>(v);
    v += dpp_move_f64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ double of_lane_f64(double v, int lane) {
    const u64 b = (u64)__double_as_longlong(v);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane), lo = (uint32_t)__builtin_amdgcn_readlane((int)b, lane);
    return __longlong_as_double((long long)((u64)hi << 32 | lo));
}
__device__ __forceinline__ double wave_sum_f64(double v) { return of_lane_f64(wave_iscan_f64(v), 63); }

// Sums of kVerifyChunk entries: sums[i][chunk] = {rest, full}.  A workgroup per request and C chunks; that of chunk 0 leaves the
// verdict, and all of the answer but the drawn token.  128 requests over 128,256 entries in 32 bits take 22 us: 105 MB
// (a row of p for each, one of q for the 60 % that had a token rejected; the others' q is not read), 4.8 TB/s, where a reading alone reaches
// 5.7 -- memory, and the chain offset -> token -> its probabilities in front of the first wide load.  One request takes 4 us, that chain
// and its row.  (Each workgroup works the verdict out for
// itself: a launch of its own for it would cost as much as the chain.)  Where there are more workgroups than the GPU holds at once,
// three chunks share that chain; one / three, us of both launches: 128 requests in 32 bits 26.0 / 25.1, in 16 bits 23.1 / 21.1, 1,024 in
// 16 bits 136 / 102, 2,000 over 32,000 entries 88 / 75, but 64 requests in 32 bits 17.6 / 19.1.
constexpr uint64_t kVerifyMany = 6144;
template <class T, int C>
__global__ __launch_bounds__(kVerifyThreads) void verify_sum_kernel(VerifyArgs A, uint64_t chunks, double2* sums, Verdict* verdicts) {
    __shared__ double2 tmp[C][kVerifyThreads / 64];
    const uint64_t groups = (chunks + C - 1) / C;
    for (uint64_t g = blockIdx.x; g < A.n * groups; g += gridDim.x) {
        const uint64_t i = g / groups, c = (g - i * groups) * C;
        const Verdict R = verdict_of<T>(A, i);
        double sr[C], sf[C];
#pragma unroll
        for (int x = 0; x < C; x++) {
            sr[x] = sf[x] = 0;
            const uint64_t col = (c + x) * kVerifyChunk + (uint64_t)threadIdx.x * 8;
            if (R.state != kBadRequest && col < A.vocab) {
                double rest[8], full[8];
                weights8<T>(A, R, col, rest, full);
#pragma unroll
                for (int j = 0; j < 8; j++) { sr[x] += rest[j]; sf[x] += full[j]; }
            }
        }
#pragma unroll
        for (int x = 0; x < C; x++) {
            const double wr = wave_sum_f64(sr[x]), wf = wave_sum_f64(sf[x]);
            if (lane_id() == 0) tmp[x][wave_id()] = make_double2(wr, wf);
        }
        __syncthreads();
        if (threadIdx.x < C && c + threadIdx.x < chunks) {
            double2 s = tmp[threadIdx.x][0];
            for (int w = 1; w < kVerifyThreads / 64; w++) { s.x += tmp[threadIdx.x][w].x; s.y += tmp[threadIdx.x][w].y; }
            sums[i * chunks + c + threadIdx.x] = s;
        }
        if (c == 0) {
            int32_t* out = A.out + i * (A.max_draft + 1ull);
            for (uint32_t j = threadIdx.x; j <= A.max_draft; j += kVerifyThreads) out[j] = R.state != kBadRequest && j < R.a ? A.draft[R.q_row - R.a + j] : -1;
            if (threadIdx.x == 0) {
                A.accepted[i] = R.state == kBadRequest ? -1 : (int32_t)R.a;
                verdicts[i] = R;
            }
        }
        __syncthreads();
    }
}

// A workgroup per request: the chunk the border falls into (every wave finds it by itself, 64 chunks at a time), then the entry.
// What bounds it is the chain of loads -- verdict and sums, then the chunk's entries -- so nothing else is on the way: 4.4 us for 128
// requests over 128,256 entries.  With the verdict worked out again and the chunks walked by one thread it took 21 us, with an atomic
// from every lane that has found an entry, instead of one from each wave, 8 us.
template <class T>
__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(VerifyArgs A, uint64_t chunks, const double2* sums, const Verdict* verdicts) {
    __shared__ double tmp[kVerifyThreads / 64];
    __shared__ int s_token, s_last;
    const int lane = lane_id();
    for (uint64_t i = blockIdx.x; i < A.n; i += gridDim.x) {
        const double2* S = sums + i * chunks;
        Verdict R = verdicts[i];
        if (!verdict_within(A, R)) R.state = kBadRequest;
        const double u = (double)A.u_draw[i];
        const double2 first = (uint64_t)lane < chunks ? S[lane] : make_double2(0, 0);   // (most vocabularies have no more chunks)
        if (threadIdx.x == 0) { s_token = 0x7FFFFFFF; s_last = -1; }
        double2 mine2 = first;
        for (uint64_t c = 64 + lane; c < chunks; c += 64) { const double2 w = S[c]; mine2.x += w.x; mine2.y += w.y; }
        const double rest = wave_sum_f64(mine2.x), full = wave_sum_f64(mine2.y);
        const bool use_rest = R.state == kDrawRest && rest > 0;
        const double border = u * (use_rest ? rest : full);
        long long at = -1, last = -1;
        double before = 0, before_last = 0, run = 0;
        for (uint64_t c0 = 0; c0 < chunks && at < 0; c0 += 64) {
            const uint64_t c = c0 + lane;
            const double2 s = c0 == 0 ? first : c < chunks ? S[c] : make_double2(0, 0);
            const double w = use_rest ? s.x : s.y, inc = run + wave_iscan_f64(w);
            const u64 some = __ballot(w > 0), over = __ballot(w > 0 && inc > border);
            if (some) {
                const int f = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
                const double b = of_lane_f64(inc - w, f);
                if (over) { at = (long long)c0 + f; before = b; } else { last = (long long)c0 + f; before_last = b; }
            }
            run = of_lane_f64(inc, 63);
        }
        // (a border that rounding has put behind all sums falls into the last chunk with weight)
        if (at < 0) { at = last; before = before_last; }
        double w8[8], mine = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) w8[j] = 0;
        const uint64_t col = (uint64_t)(at < 0 ? 0 : at) * kVerifyChunk + (uint64_t)threadIdx.x * 8;
        if (R.state != kBadRequest && at >= 0 && col < A.vocab) {
            double other[8];
            weights8<T>(A, R, col, w8, other);
#pragma unroll
            for (int j = 0; j < 8; j++) { if (!use_rest) w8[j] = other[j]; mine += w8[j]; }
        }
        const double inc = wave_iscan_f64(mine);
        if (lane == 63) tmp[wave_id()] = inc;
        __syncthreads();
        double sum = before;
        for (int w = 0; w < wave_id(); w++) sum += tmp[w];
        sum += inc - mine;
        int found = 0x7FFFFFFF, mine_last = -1;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            sum += w8[j];
            if (w8[j] > 0) {
                mine_last = (int)(col + j);
                if (sum > border && found == 0x7FFFFFFF) found = mine_last;
            }
        }
        // columns ascend with the lanes: a wave's first found entry is its first lane's, its last entry with weight its last lane's
        const u64 any_found = __ballot(found != 0x7FFFFFFF), any_last = __ballot(mine_last >= 0);
        if (any_found && lane == __builtin_ctzll(any_found)) atomicMin(&s_token, found);
        if (any_last && lane == 63 - __builtin_clzll(any_last)) atomicMax(&s_last, mine_last);
        __syncthreads();
        if (threadIdx.x == 0 && R.state != kBadRequest) A.out[i * (A.max_draft + 1ull) + R.a] = s_token != 0x7FFFFFFF ? s_token : s_last;
        __syncthreads();
    }
}

}  // namespace

hipError_t launch_verify(const VerifyArgs& A, hipStream_t stream) {
    if (A.n == 0) return hipSuccess;
    const VerifyWork W = verify_work(A.n, A.vocab);
    double2* sums = (double2*)((uint8_t*)A.work + W.sums);
    Verdict* verdicts = (Verdict*)((uint8_t*)A.work + W.verdicts);
    return with_dtype(A.dtype, [&](auto t) {
        typedef decltype(t) T;
        const bool many = W.chunks >= 3 && A.n * W.chunks >= kVerifyMany;
        hipError_t e = launch(many ? verify_sum_kernel<T, 3> : verify_sum_kernel<T, 1>, capped(A.n * (many ? (W.chunks + 2) / 3 : W.chunks)), kVerifyThreads, stream, A,
                              W.chunks, sums, verdicts);
        if (e != hipSuccess) return e;
        return launch(verify_draw_kernel<T>, capped(A.n), kVerifyThreads, stream, A, W.chunks, (const double2*)sums, (const Verdict*)verdicts);
    });
}

}  // namespace l3
