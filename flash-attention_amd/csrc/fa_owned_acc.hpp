// Accumulator registers named literally in instruction strings (see fa_fwd_w64_kernel.hpp for why and for the rules): the
// pieces that several kernels share.
#pragma once
#include "fa_fwd_kernel.hpp"

namespace fa {

// Wait states between the last MFMA on an accumulator and a v_accvgpr_read of it.
__device__ __forceinline__ void acc_fence() { asm volatile("s_nop 15\n\ts_nop 3"); }
template <int R>
__device__ __forceinline__ float acc_get() {
    float x;
    asm volatile("v_accvgpr_read_b32 %0, a[%1]" : "=v"(x) : "n"(R));
    return x;
}
template <int R>
__device__ __forceinline__ void acc_put(float x) {
    asm volatile("v_accvgpr_write_b32 a[%1], %0" : : "v"(x), "n"(R));
}
// Makes the kernel descriptor allocate a[0:31] only (D = 64: the whole accumulator).  With several waves per SIMD a
// wave's architectural and accumulator registers come out of one budget: 128 + 32 lets three workgroups share a CU.
__device__ __forceinline__ void acc_reserve32() {
    asm volatile("" : : : "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", "a14", "a15",
                 "a16", "a17", "a18", "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", "a27", "a28", "a29", "a30", "a31");
}
__device__ __forceinline__ void acc_reserve64() {
    asm volatile("" : : : "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", "a14", "a15",
                 "a16", "a17", "a18", "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", "a27", "a28", "a29", "a30", "a31",
                 "a32", "a33", "a34", "a35", "a36", "a37", "a38", "a39", "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47",
                 "a48", "a49", "a50", "a51", "a52", "a53", "a54", "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63");
}
// a[LO : LO+15] = 0 through the matrix pipe; a[BASE : BASE+N-1] *= alpha through the vector ALU (rare: the rescale).
template <int LO>
__device__ __forceinline__ void acc_zero16() {
    half8 z = {};
    asm volatile("s_nop 3" : "+v"(z));  // wait states between the vector writes of z and the MFMA reading it
    asm volatile("v_mfma_f32_32x32x16_f16 a[%1:%2], %0, %0, 0" : : "v"(z), "n"(LO), "n"(LO + 15));
}
template <int BASE, int N>
__device__ __forceinline__ void acc_scale_n(float alpha) {
    acc_fence();
    static_for<N>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        acc_put<BASE + i>(acc_get<BASE + i>() * alpha);
    });
}

// (a[0:127]: D = 256)
__device__ __forceinline__ void acc_reserve128() {
    acc_reserve64();
    asm volatile("" : : : "a64", "a65", "a66", "a67", "a68", "a69", "a70", "a71", "a72", "a73", "a74", "a75", "a76", "a77", "a78", "a79", "a80",
                 "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", "a91", "a92", "a93", "a94", "a95", "a96", "a97", "a98",
                 "a99", "a100", "a101", "a102", "a103", "a104", "a105", "a106", "a107", "a108", "a109", "a110", "a111", "a112", "a113", "a114",
                 "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", "a124", "a125", "a126", "a127");
}

}  // namespace fa
