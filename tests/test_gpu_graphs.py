"""GPU: captured graphs give on every replay what the eager calls give, library reductions included."""
import copy
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


def batch(n, gen):
    p = torch.rand(n, 192, device="cuda", generator=gen)
    won = torch.randint(0, 2, (n,), device="cuda", generator=gen)
    return ((torch.rand(n, 3, 8, 8, device="cuda", generator=gen) > 0.7).float(), p / p.sum(1, keepdim=True), torch.stack((won, 1 - won), 1).float())


@pytest.mark.parametrize("n", [1024, 4096])
@pytest.mark.parametrize("dtype", [None, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("fused", [False, True], ids=["plain", "fused"])
def test_gradients_of_every_replay_are_the_eager_ones(n, dtype, fused):
    """Four replays of a captured step's forward and backward pass, with eager work and synchronisation between them: every
    parameter's gradient, each of them against eager calls from the same weights.  The two sides make the same calls; sums whose
    order is not fixed (the convolutions' weight gradients) end rounded to the type: half a step of each value, 2^-8 of the norm
    in bfloat16 and, for a few thousand float32 terms, 1e-4."""
    from alphazero_amd import distributed
    from alphazero_amd.model import AlphaZeroNet
    torch.manual_seed(1)
    model = AlphaZeroNet(num_blocks=2, num_filters=32).cuda().use_fused_ops(fused)
    optimizer = torch.optim.Adam(model.parameters(), lr=1e-3)
    gen = torch.Generator("cuda").manual_seed(2)
    step = distributed.GraphedTrainStep(model, optimizer, n, autocast_dtype=dtype)
    for _ in range(4):                                                 # three eager steps, then the captures and one replay
        step(*batch(n, gen))
    for replay in range(4):
        for held, new in zip((step.states, step.pis, step.wls), batch(n, gen)):
            held.copy_(new)
        twin = copy.deepcopy(model).train()
        for p in twin.parameters():
            p.grad = None
        step.sums.zero_()
        step.graph_a.replay()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = distributed.losses(twin, step.states, step.pis, step.wls, dtype)
            want[0].backward()
        torch.cuda.synchronize()
        for got, v in zip(step.sums.tolist(), want):
            assert abs(got - float(v.detach())) <= 1e-3 * abs(float(v.detach())), replay
        for (name, a), b in zip(model.named_parameters(), twin.parameters()):
            assert float((a.grad - b.grad).norm()) <= (1e-4 if dtype is None else 2.0 ** -8) * float(b.grad.norm()), (replay, name)


def memset_nodes(graph):
    """How many memset nodes az_graph_fill_by_kernels finds (and replaces)."""
    from alphazero_amd import _lib
    found = C.c_int32()
    _lib.check(_lib.lib().az_graph_fill_by_kernels(graph.raw_cuda_graph(), C.byref(found)))
    return found.value


def test_memset_nodes_are_replaced_where_they_stand():
    """A column sum of many rows between kernels that write its input and read its output: replays follow the input, and no
    memset node is left."""
    from alphazero_amd.distributed import capture
    gen = torch.Generator("cuda").manual_seed(3)
    x = torch.zeros(4096, 130, dtype=torch.bfloat16, device="cuda")
    source, out = torch.zeros_like(x), torch.zeros(130, device="cuda")

    def work():
        x.copy_(source)
        out.copy_(x.sum(0).float() * 2)
    work()                                                             # whatever a first call sets up
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        work()
    assert memset_nodes(graph) >= 0 and memset_nodes(graph) == 0
    captured = capture(work)
    for _ in range(4):
        source.copy_(torch.randn(x.shape, device="cuda", generator=gen).to(x.dtype))
        captured.replay()
        torch.cuda.synchronize()
        got = out.clone()
        work()
        torch.cuda.synchronize()
        assert torch.equal(got, out)


@pytest.mark.parametrize("width, height, pitch, size, value", [(1, 1, 1, 1, 7), (1000, 1, 1000, 1, 255), (1001, 1, 0, 1, 0x7F), (64, 1, 0, 1, 0xAB), (333, 1, 0, 4, 0xDEADBEEF),
                                                               (77, 1, 0, 2, 0xBEEF), (10, 5, 64, 1, 3), (3, 7, 20, 4, 1), (1 << 20, 1, 0, 4, 2)])
def test_every_form_of_a_memset_node(width, height, pitch, size, value):
    """A graph made by hand: what the replacing kernel writes, and nothing else, by bytes."""
    from alphazero_amd import _lib
    L = _lib.lib()
    hip = C.CDLL("libamdhip64.so", mode=C.RTLD_GLOBAL) if not hasattr(L, "hipGraphCreate") else L

    class Params(C.Structure):
        _fields_ = [("dst", C.c_void_p), ("elementSize", C.c_uint), ("height", C.c_size_t), ("pitch", C.c_size_t), ("value", C.c_uint), ("width", C.c_size_t)]
    span = width * size if height == 1 else (height - 1) * pitch + width * size
    held = torch.full((span + 32,), 0xAA, dtype=torch.uint8, device="cuda")
    graph, node = C.c_void_p(), C.c_void_p()
    assert hip.hipGraphCreate(C.byref(graph), 0) == 0
    p = Params(held.data_ptr() + 16, size, height, pitch or width * size, value, width)
    assert hip.hipGraphAddMemsetNode(C.byref(node), graph, None, C.c_size_t(0), C.byref(p)) == 0
    found = C.c_int32()
    _lib.check(L.az_graph_fill_by_kernels(graph, C.byref(found)))
    assert found.value == 1
    run = C.c_void_p()
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    assert hip.hipGraphLaunch(run, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    want = torch.full((span + 32,), 0xAA, dtype=torch.uint8)
    word = torch.tensor(list(value.to_bytes(4, "little"))[:size], dtype=torch.uint8)
    for row in range(height):
        at = 16 + row * pitch
        want[at:at + width * size] = word.repeat(width)
    assert torch.equal(held.cpu(), want)
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
