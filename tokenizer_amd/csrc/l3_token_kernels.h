// l3_token_kernels.h -- launch interface of the operators on token ids, and what their translation units share.
#pragma once
#include <hip/hip_runtime.h>

#include "l3_token_ops.h"

namespace l3 {

// Queue the operator's kernels on `stream`; nothing is synchronised, allocated or kept.  The arguments have been checked.
hipError_t launch_embed(const EmbedArgs& A, hipStream_t stream);
hipError_t launch_embed_grad(const EmbedGradArgs& A, hipStream_t stream);
hipError_t launch_cache_slots(const CacheArgs& A, hipStream_t stream);
hipError_t launch_cache_trim(const CacheArgs& A, hipStream_t stream);
hipError_t launch_verify(const VerifyArgs& A, hipStream_t stream);

namespace {

// A launch whose error is its own: hipGetLastError would hand out (and clear) what another library's call left behind.
template <class... P>
hipError_t launch(void (*kernel)(P...), uint64_t blocks, uint32_t threads, hipStream_t stream, P... args) {
    if (blocks * threads >= 1ull << 32) return hipErrorInvalidConfiguration;   // (the runtime cuts such a grid short without a word)
    void* a[] = {(void*)&args...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3((uint32_t)blocks), dim3(threads), a, 0, stream);
}
// For kernels that walk their work with the grid's stride.
constexpr uint64_t kMaxBlocks = 1u << 21;
inline uint64_t capped(uint64_t blocks) { return blocks < kMaxBlocks ? blocks : kMaxBlocks; }

// f(T{}) for the element type of a code that has been checked
template <class F>
hipError_t with_dtype(int code, F f) {
    return code == kF32 ? f(float()) : code == kF16 ? f(_Float16()) : f((__bf16)0.f);
}

// N neighbouring elements, aligned like one of them: any row start and stride is fine, gfx950 takes unaligned 16-byte accesses.
template <class T, int N = 8> struct Few {
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    typedef float F __attribute__((ext_vector_type(N)));
};
template <class T> using Eight = Few<T, 8>;
typedef float F8 __attribute__((ext_vector_type(8)));
template <int N = 8, class T>
__device__ __forceinline__ typename Few<T, N>::V load8(const T* p) { return *reinterpret_cast<const typename Few<T, N>::V*>(p); }
template <class V>
__device__ __forceinline__ F8 to_f8(V v) { return __builtin_convertvector(v, F8); }
// Stores round to nearest, ties to even.
template <int N = 8, class T>
__device__ __forceinline__ void store8(T* p, typename Few<T, N>::F v) {
    *reinterpret_cast<typename Few<T, N>::V*>(p) = __builtin_convertvector(v, typename Few<T, N>::V);
}
// The same for data that is used once: it need not stay in the caches.  (Stores: 16 bytes a lane, neighbouring lanes side by side --
// what a wave's store leaves open of a cache line is not put together with the next store's.)
template <int N = 8, class T>
__device__ __forceinline__ typename Few<T, N>::V load8_once(const T* p) { return __builtin_nontemporal_load(reinterpret_cast<const typename Few<T, N>::V*>(p)); }
template <int N = 8, class T>
__device__ __forceinline__ void store8_once(T* p, typename Few<T, N>::F v) {
    __builtin_nontemporal_store(__builtin_convertvector(v, typename Few<T, N>::V), reinterpret_cast<typename Few<T, N>::V*>(p));
}

}  // namespace

}  // namespace l3
