// Captured HIP graphs without memset nodes.
//
// Library calls clear their semaphores with hipMemsetAsync (a sum over many rows does, as the gradient of a linear layer's
// bias), and a capture records that as a memset node.  Such nodes have given wrong results on every replay after the
// first on this hardware: at 1024 rows in bfloat16 a bias gradient was off by a factor of 17, or infinite.  So each is
// replaced by a kernel that writes the same bytes, between the same neighbours, before the graph is instantiated.
#include <exception>
#include <vector>

#include "az_common.h"

namespace az {

// height rows of width elements of SIZE bytes, pitch bytes apart
template <typename T>
__global__ __launch_bounds__(256) void k_graph_fill(char* dst, uint64_t pitch, uint64_t width, uint64_t height, T value) {
    const uint64_t n = width * height;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = height == 1 ? 0 : i / width;
        ((T*)(dst + row * pitch))[i - row * width] = value;
    }
}

template <typename T>
static hipError_t add_fill(hipGraphNode_t* node, hipGraph_t graph, const std::vector<hipGraphNode_t>& after, const hipMemsetParams& m) {
    char* dst = (char*)m.dst;
    uint64_t pitch = m.pitch, width = m.width, height = m.height;
    T value = (T)m.value;
    void* args[] = {&dst, &pitch, &width, &height, &value};
    const uint64_t blocks = (width * height + 255) / 256;
    hipKernelNodeParams k = {};
    k.func = (void*)k_graph_fill<T>;
    k.gridDim = dim3((uint32_t)(blocks < 1 ? 1 : blocks < 4096 ? blocks : 4096));
    k.blockDim = dim3(256);
    k.kernelParams = args;
    return hipGraphAddKernelNode(node, graph, after.data(), after.size(), &k);
}

static int fill_by_kernels(hipGraph_t graph, int32_t* replaced) {
    size_t n = 0;
    AZ_HIP(hipGraphGetNodes(graph, nullptr, &n));
    std::vector<hipGraphNode_t> nodes(n);
    if (n) AZ_HIP(hipGraphGetNodes(graph, nodes.data(), &n));
    for (hipGraphNode_t node : nodes) {
        hipGraphNodeType type;
        AZ_HIP(hipGraphNodeGetType(node, &type));
        if (type == hipGraphNodeTypeGraph) {
            hipGraph_t child;
            AZ_HIP(hipGraphChildGraphNodeGetGraph(node, &child));
            const int rc = fill_by_kernels(child, replaced);
            if (rc != AZ_OK) return rc;
        }
        if (type != hipGraphNodeTypeMemset) continue;
        hipMemsetParams m = {};
        AZ_HIP(hipGraphMemsetNodeGetParams(node, &m));
        if (m.elementSize != 1 && m.elementSize != 2 && m.elementSize != 4)
            AZ_FAIL(AZ_ERR_STATE, "a memset node of %u-byte elements", m.elementSize);
        size_t before = 0, behind = 0;
        AZ_HIP(hipGraphNodeGetDependencies(node, nullptr, &before));
        std::vector<hipGraphNode_t> from(before);
        if (before) AZ_HIP(hipGraphNodeGetDependencies(node, from.data(), &before));
        AZ_HIP(hipGraphNodeGetDependentNodes(node, nullptr, &behind));
        std::vector<hipGraphNode_t> to(behind);
        if (behind) AZ_HIP(hipGraphNodeGetDependentNodes(node, to.data(), &behind));
        hipGraphNode_t fill;
        if (m.elementSize == 1 && m.height == 1 && (uintptr_t)m.dst % 4 == 0 && m.width % 4 == 0) {      // by words
            m.elementSize = 4;
            m.width /= 4;
            m.value = (m.value & 0xFF) * 0x01010101u;
        }
        if (m.elementSize == 1) AZ_HIP(add_fill<uint8_t>(&fill, graph, from, m));
        else if (m.elementSize == 2) AZ_HIP(add_fill<uint16_t>(&fill, graph, from, m));
        else AZ_HIP(add_fill<uint32_t>(&fill, graph, from, m));
        for (hipGraphNode_t& next : to) AZ_HIP(hipGraphAddDependencies(graph, &fill, &next, 1));
        for (hipGraphNode_t& previous : from) AZ_HIP(hipGraphRemoveDependencies(graph, &previous, &node, 1));
        for (hipGraphNode_t& next : to) AZ_HIP(hipGraphRemoveDependencies(graph, &node, &next, 1));
        AZ_HIP(hipGraphDestroyNode(node));
        ++*replaced;
    }
    return AZ_OK;
}

}  // namespace az

extern "C" int az_graph_fill_by_kernels(void* graph, int32_t* replaced_host) try {
    AZ_CHECK_ARG(graph && replaced_host, "az_graph_fill_by_kernels: null argument");
    *replaced_host = 0;
    return az::fill_by_kernels((hipGraph_t)graph, replaced_host);
} catch (const std::exception& e) {
    AZ_FAIL(AZ_ERR_STATE, "az_graph_fill_by_kernels: %s", e.what());
}
