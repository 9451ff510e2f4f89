// Shared by the translation units of the library; not part of the public ABI.
#pragma once

#include <cstdint>

#include <cuda.h>
#include <cuda_runtime.h>

namespace ckl {

// Records `fmt` as the calling thread's last error (what ckl_last_error() returns) and
// returns `code`, so a failing path can `return set_error(CKL_ERR_..., "...", ...)`.
int set_error(int code, const char* fmt, ...);

// What the entry points share of the current device's state.  device_view creates the state on
// a device's first use (a small cudaMalloc) and fails with CKL_ERR_UNSUPPORTED off sm_100.
struct DeviceView {
    int device;
    int sm_count;
    int max_pairs;         // CTA pairs that can be resident at once
    unsigned int* status;  // 4 words on the device, read by ckl_device_status
};
int device_view(DeviceView* out);

// Encodes a TMA descriptor of a stack of row-major matrices: `inner` columns, `outer` rows of
// `pitch` elements, `depth` matrices `stack` elements apart (depth 0: one matrix, a 2-D map).
// 64- or 128-byte swizzle, as wide as the box; zeros outside.  An empty tensor gives an unused,
// zeroed descriptor.
int encode_operand(CUtensorMap* map, int dtype, const void* base, uint64_t inner, uint64_t outer,
                   uint64_t pitch, uint64_t depth, uint64_t stack, uint32_t box_inner,
                   uint32_t box_outer);

// Largest count of rows, columns, tokens or slots of the routed operators: their kernels round such
// counts up and step past them in 32 bits by less than the rest.
constexpr int kMaxExtent = 0x7fffffff - 4095;

// Launches a kernel as a programmatic dependent: it may be set up while the kernel before it on
// the stream finishes, and waits for that one itself before it touches memory.
template <typename... Params, typename... Args>
inline cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t smem,
                                    int cluster, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The wait fault armed by ckl_test_arm_wait_fault for the calling thread (kind 0: none); disarms it.
int take_wait_fault(unsigned long long* limit_ns);

}  // namespace ckl
