"""Memory that an operator made itself, when the operator is dropped while its call on another stream has not run yet."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv import Served

pytestmark = pytest.mark.gpu


def _product(F):
    m, n, k = 64, 512, 8192
    (a, sa), (b, _) = F.new_rows(m, k), F.new_rows(n, k)
    op = F.Fp8Matmul(a, sa, b, torch.zeros(n // 128, k // 128, device="cuda"), torch.zeros(m, n, dtype=torch.bfloat16, device="cuda"))
    return op, [op.workspace]


def _plan(F):
    op = F.ExpertPlan(torch.zeros(1024, 8, dtype=torch.int32, device="cuda"), 128)
    return op, [op.workspace, op.group_start, op.tokens, op.slots]


def _attention(F):
    from stark_amd import kv
    s = Served(kv, 20, [(1, 6000), (1, 4000)], 8, 2, 128, 64, 16, "bf16")
    op = s.operator()
    op.served = s
    return op, [op.workspace]


def _kv_plan(F):
    from stark_amd import kv
    i = torch.int32
    op = kv.KvPlan(torch.zeros(4, dtype=i, device="cuda"), torch.ones(4, dtype=i, device="cuda"), torch.arange(8, dtype=i, device="cuda"),
                   torch.full((1,), 8, dtype=i, device="cuda"), torch.full((4, 2), -1, dtype=i, device="cuda"), 16, 3000)
    return op, [op.slots, op.positions, op.kv_lengths]


@pytest.fixture(scope="module")
def F(qmm):
    from stark_amd import fp8
    return fp8


def _ranges(tensors):
    return [(t.data_ptr(), t.numel() * t.element_size()) for t in tensors]


def _meets(places, busy=lambda: True):
    """Tensors of the places' sizes, each until the allocator has no free memory left for it: whether one that was made while the
    stream was busy lies in a place."""
    got, counted = [], 0
    for _, size in places:
        before = torch.cuda.memory_reserved()
        while torch.cuda.memory_reserved() == before:  # (the last one, of new memory, may wait for the device)
            got.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
            if busy():
                counted = len(got)
    assert counted
    return any(p < q + m and q < p + n for p, n in places for q, m in _ranges(got[:counted]))


@pytest.mark.parametrize("how", ["given", "current", "handle first"])
@pytest.mark.parametrize("make", [_product, _plan, _attention, _kv_plan])
def test_memory_waits_for_the_stream(F, make, how):
    """The call waits behind some tens of ms of other work on its stream; what is allocated meanwhile is not the operator's memory."""
    x = torch.randn(8192, 8192, dtype=torch.bfloat16, device="cuda")
    y = torch.empty_like(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.mm(x, x, out=y)  # the library's own start
    op, made = make(F)
    assert all(t is not None for t in made)
    places = _ranges(made)[:1]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(60):
            torch.mm(x, x, out=y)
        if how == "current":
            op.encode()
    if how == "handle first":  # of which torch knows nothing
        op.encode(stream=side.cuda_stream)
    if how != "current":
        op.encode(stream=side)
    del op, made
    assert not _meets(places, lambda: not side.query())
    torch.cuda.synchronize()


@pytest.mark.parametrize("make", [_product, _plan, _attention, _kv_plan])
def test_memory_of_one_stream_returns_at_once(F, make):
    """The control of the test above: on the stream that an operator was made on, its memory is the next tensors'."""
    op, made = make(F)
    places = _ranges(made)
    op.encode()
    del op, made
    assert _meets(places)
    torch.cuda.synchronize()


def test_a_captured_call_on_another_stream(F):
    """A capture's stream is another one: the operator lives, its call replays."""
    ids = torch.from_numpy(np.random.default_rng(1).integers(0, 128, (1024, 8)).astype(np.int32)).cuda()
    op = F.ExpertPlan(ids, 128)
    op.encode()
    torch.cuda.synchronize()
    want = op.slots.clone()
    g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=stream):
        op.encode()
    for _ in range(3):
        op.slots.fill_(-7)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(op.slots, want)
