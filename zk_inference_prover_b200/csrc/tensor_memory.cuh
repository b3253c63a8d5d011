// What kernels that multiply on the tensor cores' own memory (tcgen05) share: commits, fences, and moves between that memory and registers.
#pragma once
#include <cstdint>

namespace zk {

// The barrier gets an arrival when the products issued so far are done.
__device__ __forceinline__ void products_done(uint32_t bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#define R8(x, o) "=r"(x[o]), "=r"(x[o + 1]), "=r"(x[o + 2]), "=r"(x[o + 3]), "=r"(x[o + 4]), "=r"(x[o + 5]), "=r"(x[o + 6]), "=r"(x[o + 7])
#define W8(x, o) "r"(x[o]), "r"(x[o + 1]), "r"(x[o + 2]), "r"(x[o + 3]), "r"(x[o + 4]), "r"(x[o + 5]), "r"(x[o + 6]), "r"(x[o + 7])
// 32, 16 or 8 columns of this thread's row; they are there after tmem_loaded, which names them so that nothing that uses them is moved before it.
#define RW8(x, o) "+r"(x[o]), "+r"(x[o + 1]), "+r"(x[o + 2]), "+r"(x[o + 3]), "+r"(x[o + 4]), "+r"(x[o + 5]), "+r"(x[o + 6]), "+r"(x[o + 7])
__device__ __forceinline__ void tmem_loaded(uint32_t (&x)[32]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : RW8(x, 0), RW8(x, 8), RW8(x, 16), RW8(x, 24)::"memory"); }
__device__ __forceinline__ void tmem_loaded(uint32_t (&x)[16]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : RW8(x, 0), RW8(x, 8)::"memory"); }
__device__ __forceinline__ void tmem_loaded(uint32_t (&x)[8]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : RW8(x, 0)::"memory"); }
#undef RW8
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t* x) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : R8(x, 0), R8(x, 8), R8(x, 16), R8(x, 24) : "r"(at));
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t* x) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];" : R8(x, 0), R8(x, 8) : "r"(at));
}
__device__ __forceinline__ void tmem_load8(uint32_t at, uint32_t* x) { asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : R8(x, 0) : "r"(at)); }
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t* x) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
                 W8(x, 0), W8(x, 8), W8(x, 16), W8(x, 24) : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t at, const uint32_t* x) { asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), W8(x, 0) : "memory"); }
// The same word to sixteen columns of this thread's row.
__device__ __forceinline__ void tmem_fill16(uint32_t at, uint32_t w) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1};" ::"r"(at), "r"(w) : "memory");
}
#undef R8
#undef W8

__device__ __forceinline__ uint64_t two_words(uint32_t a, uint32_t b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t bar_of(const unsigned long long& b) { return (uint32_t)__cvta_generic_to_shared(&b); }
// Two 32-bit floats at once.
__device__ __forceinline__ uint64_t both(float a, float b) { return two_words(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ uint64_t add_both(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul_both(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma_both(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float first_of(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float second_of(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }

}  // namespace zk
