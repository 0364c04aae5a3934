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
    void* a[] = {(void*)&args...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3((uint32_t)blocks), dim3(threads), a, 0, stream);
}
// A grid has at most 2^32 - 1 work-items; every kernel here walks its work with the grid's stride, so a cap costs nothing.
constexpr uint64_t kMaxBlocks = 1u << 21;
inline uint64_t capped(uint64_t blocks) { return blocks < kMaxBlocks ? blocks : kMaxBlocks; }

// f(T{}) for the element type of a code that has been checked
template <class F>
hipError_t with_dtype(int code, F f) {
    return code == kF32 ? f(float()) : code == kF16 ? f(_Float16()) : f((__bf16)0.f);
}

// Eight neighbouring elements, aligned like one of them: any row start and stride is fine, gfx950 takes unaligned 16-byte accesses.
template <class T> struct Eight {
    typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
typedef float F8 __attribute__((ext_vector_type(8)));
template <class T>
__device__ __forceinline__ typename Eight<T>::V load8(const T* p) { return *reinterpret_cast<const typename Eight<T>::V*>(p); }
// The same for data that is used once: it need not stay in the caches.
template <class T>
__device__ __forceinline__ typename Eight<T>::V load8_once(const T* p) { return __builtin_nontemporal_load(reinterpret_cast<const typename Eight<T>::V*>(p)); }
template <class T>
__device__ __forceinline__ void store8_once(T* p, F8 v) {
    __builtin_nontemporal_store(__builtin_convertvector(v, typename Eight<T>::V), reinterpret_cast<typename Eight<T>::V*>(p));
}
template <class V>
__device__ __forceinline__ F8 to_f8(V v) { return __builtin_convertvector(v, F8); }
template <class T>
__device__ __forceinline__ void store8(T* p, F8 v) {   // rounded to nearest, ties to even
    *reinterpret_cast<typename Eight<T>::V*>(p) = __builtin_convertvector(v, typename Eight<T>::V);
}

}  // namespace

}  // namespace l3
