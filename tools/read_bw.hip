// Development aid: what does a read-only stream reach on this GPU?  Workgroups of 256 threads read disjoint contiguous
// chunks (as the decode cross-attention does with its K/V ranges), U 16-byte loads per thread in flight, plain or
// non-temporal; the sum goes to one float per workgroup so nothing is optimised away.
//   hipcc --offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops -O3 tools/read_bw.hip -o tools/read_bw
#include <hip/hip_runtime.h>
#include <cstdio>
#include <cstdlib>
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <int U, bool NT>
__global__ __launch_bounds__(256) void read_kernel(const u32x4* __restrict__ src, float* __restrict__ out, long chunk16) {
    // chunk16: 16-byte pieces per workgroup, a multiple of 256 * U
    const u32x4* p = src + (long)blockIdx.x * chunk16 + threadIdx.x;
    unsigned acc = 0;
    for (long i = 0; i < chunk16; i += 256 * U) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = NT ? __builtin_nontemporal_load(p + i + u * 256) : p[i + u * 256];
#pragma unroll
        for (int u = 0; u < U; ++u) acc += v[u][0] ^ v[u][1] ^ v[u][2] ^ v[u][3];
    }
    if (acc == 0x12345678u) out[blockIdx.x] = 1.f;      // practically never: keeps the loads alive
}

template <int U, bool NT>
static void run(const u32x4* src, float* out, size_t bytes, long chunk_bytes, int lds_pad, const char* name) {
    const long chunk16 = chunk_bytes / 16;
    const int grid = (int)(bytes / chunk_bytes);
    hipEvent_t e0, e1; (void)hipEventCreate(&e0); (void)hipEventCreate(&e1);
    hipLaunchKernelGGL((read_kernel<U, NT>), dim3(grid), dim3(256), lds_pad, 0, src, out, chunk16);
    (void)hipEventRecord(e0, 0);
    for (int i = 0; i < 10; ++i) hipLaunchKernelGGL((read_kernel<U, NT>), dim3(grid), dim3(256), lds_pad, 0, src, out, chunk16);
    (void)hipEventRecord(e1, 0); (void)hipEventSynchronize(e1);
    float ms = 0; (void)hipEventElapsedTime(&ms, e0, e1);
    printf("%-28s chunk %6ld KB  lds %5d  grid %6d : %7.1f us %7.1f GB/s\n", name, chunk_bytes / 1024, lds_pad, grid, ms * 100, (double)grid * chunk_bytes * 10.0 / ms / 1e6);
}

int main(int argc, char** argv) {
    setvbuf(stdout, nullptr, _IONBF, 0);
    // default 6 GiB: far beyond the 256 MiB Infinity Cache; argv[1]: MiB per launch (rounded to 3 MiB)
    const size_t bytes = argc > 1 ? (size_t)atol(argv[1]) / 3 * 3 << 20 : (size_t)6 << 30;
    u32x4* src; float* out;
    if (hipMalloc(&src, bytes) != hipSuccess || hipMalloc(&out, 1 << 22) != hipSuccess) { printf("alloc failed\n"); return 1; }
    (void)hipMemset(src, 1, bytes);
    for (int lds : {0, 40000, 65536}) {
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(read_kernel<12, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 65536);
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(read_kernel<12, false>), hipFuncAttributeMaxDynamicSharedMemorySize, 65536);
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(read_kernel<4, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 65536);
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(read_kernel<8, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 65536);
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(read_kernel<16, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 65536);
        run<12, true>(src, out, bytes, 48 * 1024, lds, "12 in flight, nt");
        run<12, false>(src, out, bytes, 48 * 1024, lds, "12 in flight, plain");
        run<4, true>(src, out, bytes, 48 * 1024, lds, "4 in flight, nt");
        run<8, true>(src, out, bytes, 64 * 1024, lds, "8 in flight, nt");
        run<16, true>(src, out, bytes, 64 * 1024, lds, "16 in flight, nt");
        run<12, true>(src, out, bytes, 96 * 1024, lds, "12 in flight, nt");
        run<12, true>(src, out, bytes, 384 * 1024, lds, "12 in flight, nt");
        run<16, true>(src, out, bytes, 1024 * 1024, lds, "16 in flight, nt");
    }
    return 0;
}
