// Memset nodes of a captured graph, replaced by a fill kernel.
//
// Libraries record hipMemsetAsync into a capture where they clear workspaces and
// results (MIOpen's weight gradients, torch's reductions over many blocks). On this
// hardware such nodes write wrongly in replays after the first: the gradients of
// a captured training step (ResNet-50 of 224 x 224, 39 of these nodes) came out as
// 1e12 and NaN from the second replay on. A kernel node in the node's place, with its
// edges, does what it stands for.
//
// The fill is bound by memory: 16 bytes a thread and step, single bytes at a row's
// ends, where it starts or stops inside 16.

#include <torch/extension.h>
#include <c10/core/Device.h>
#include <c10/hip/HIPException.h>
#include <hip/hip_runtime.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <vector>

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// rows of `bytes` bytes, `pitch` apart; pattern repeats every 4 bytes from a row's
// start on
__global__ __launch_bounds__(256)
void graph_fill_kernel(char* __restrict__ dst, size_t pitch, size_t bytes,
                       size_t height, unsigned pattern) {
    const size_t step = (size_t)gridDim.x * 256;
    for (size_t row = blockIdx.y; row < height; row += gridDim.y) {
        char* const lo = dst + row * pitch;
        char* const hi = lo + bytes;
        const unsigned off = (unsigned)((uintptr_t)lo & 15);
        // the pattern as it lies from a multiple of 4 on
        const unsigned turn = (off & 3) * 8;
        const unsigned w = turn ? pattern << turn | pattern >> (32 - turn) : pattern;
        const size_t pieces = (off + bytes + 15) / 16;
        for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += step) {
            char* const p = lo - off + i * 16;
            if (p >= lo && p + 16 <= hi) {
                *reinterpret_cast<u32x4*>(p) = (u32x4){w, w, w, w};
            } else {
                for (int b = 0; b < 16; ++b)
                    if (p + b >= lo && p + b < hi)
                        p[b] = (char)(w >> (b & 3) * 8);
            }
        }
    }
}

using Nodes = std::vector<hipGraphNode_t>;

template <class F>
Nodes list_of(F&& get) {
    size_t n = 0;
    C10_HIP_CHECK(get(nullptr, &n));
    Nodes v(n);
    if (n) C10_HIP_CHECK(get(v.data(), &n));
    v.resize(n);
    return v;
}

// The graph (torch.cuda.CUDAGraph.raw_cuda_graph()) before it is instantiated; how
// many nodes were replaced.
int64_t graph_fill_nodes(uint64_t raw) {
    const hipGraph_t graph = reinterpret_cast<hipGraph_t>(raw);
    int64_t count = 0;
    for (hipGraphNode_t node : list_of([&](hipGraphNode_t* p, size_t* n) {
             return hipGraphGetNodes(graph, p, n); })) {
        hipGraphNodeType type;
        C10_HIP_CHECK(hipGraphNodeGetType(node, &type));
        TORCH_CHECK(type != hipGraphNodeTypeGraph,
                    "graph_fill_nodes: a graph within the graph");
        if (type != hipGraphNodeTypeMemset) continue;
        hipMemsetParams m;
        C10_HIP_CHECK(hipGraphMemsetNodeGetParams(node, &m));
        const unsigned es = m.elementSize;
        TORCH_CHECK(es == 1 || es == 2 || es == 4, "graph_fill_nodes: elements of ",
                    es, " bytes");
        unsigned pattern = es == 1 ? (m.value & 0xffu) * 0x01010101u
                         : es == 2 ? (m.value & 0xffffu) * 0x00010001u : m.value;
        const Nodes from = list_of([&](hipGraphNode_t* p, size_t* n) {
            return hipGraphNodeGetDependencies(node, p, n); });
        const Nodes to = list_of([&](hipGraphNode_t* p, size_t* n) {
            return hipGraphNodeGetDependentNodes(node, p, n); });
        size_t bytes = m.width * es, pitch = m.pitch, height = m.height;
        const size_t blocks = (bytes / 16 + 2 + 255) / 256;
        void* args[] = {&m.dst, &pitch, &bytes, &height, &pattern};
        hipKernelNodeParams k{};
        k.func = reinterpret_cast<void*>(&graph_fill_kernel);
        k.gridDim = dim3((unsigned)std::min<size_t>(blocks, 2048),
                         (unsigned)std::min<size_t>(std::max<size_t>(height, 1), 1024));
        k.blockDim = dim3(256);
        k.kernelParams = args;
        hipGraphNode_t fill;
        C10_HIP_CHECK(hipGraphAddKernelNode(&fill, graph, from.data(), from.size(), &k));
        for (hipGraphNode_t t : to)
            C10_HIP_CHECK(hipGraphAddDependencies(graph, &fill, &t, 1));
        C10_HIP_CHECK(hipGraphDestroyNode(node));
        ++count;
    }
    return count;
}

// Whether an autograd graph that ends in one of the tensors is alive.
bool grad_graph_alive(const std::vector<at::Tensor>& leaves) {
    return std::any_of(leaves.begin(), leaves.end(), [](const at::Tensor& t) {
        return t.is_leaf() && t.requires_grad() &&
               torch::autograd::impl::try_get_grad_accumulator(t) != nullptr;
    });
}

}  // namespace

void register_graph(pybind11::module& m) {
    m.def("graph_fill_nodes", &graph_fill_nodes,
          "memset nodes of a captured graph to fill kernels; how many");
    m.def("grad_graph_alive", &grad_graph_alive,
          "whether an autograd graph that ends in one of the tensors is alive");
}
