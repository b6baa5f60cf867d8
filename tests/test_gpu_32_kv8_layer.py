"""GPU tests of the 8-bit cache's operators together, as a layer runs them: tables, rotary positions, writer, attention, reader; eager,
captured with lengths that change at replay, on several streams, and behind one another without a wait."""
import math

import pytest
import torch

from pth_flash_attn_b200 import capi, kv8, ops
from tests.kv8_util import E4M3, check, reference

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
PAGE, GROUP, HQ, HKV, D = 32, 16, 8, 2, 128


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Layer:
    """A layer's cache and the buffers of its steps, for up to ``tokens`` tokens of ``requests`` requests."""

    def __init__(self, requests, tokens, pages, seed=0, blocks=None):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.blocks = blocks or requests * pages
        z = lambda *n, t=torch.int32: torch.zeros(n, dtype=t, device="cuda")
        self.k, self.v = (torch.full((self.blocks, PAGE, HKV, D), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
        self.ks, self.vs = (torch.full((self.blocks, PAGE // GROUP, HKV), math.nan, device="cuda") for _ in range(2))
        self.context, self.new, self.seq, self.starts = z(requests), z(requests), z(requests), z(requests + 1)
        self.table, self.slots, self.positions, self.taken = z(requests, pages), z(tokens, t=torch.int64), z(tokens, t=torch.int64), z(1)
        self.free = torch.randperm(self.blocks, generator=self.gen, device="cuda").to(torch.int32)
        self.f, self.scale = ops.rotary_frequencies(D, scaling="yarn", factor=4.0, device="cuda")
        self.q, self.key, self.value = (torch.zeros((tokens, h, D), dtype=BF16, device="cuda") for h in (HQ, HKV, HKV))
        self.q_turned, self.k_turned, self.out = torch.zeros_like(self.q), torch.zeros_like(self.key), torch.zeros_like(self.q)
        self.lse = torch.zeros((tokens, HQ), device="cuda")
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        self.ws = torch.zeros(kv8.workspace_bytes(D=D, num_sms=sms), dtype=torch.uint8, device="cuda")
        self.kept = []   # keys and values that were written, per request

    def feed(self, context, new):
        """The next step's inputs, into the same buffers."""
        self.context.copy_(_i32(context))
        self.new.copy_(_i32(new))
        for x in (self.q, self.key, self.value):
            x.copy_(torch.randn(x.shape, generator=self.gen, device="cuda"))

    def step(self, longest):
        ops.page_tables(self.context, self.new, self.free, self.table, self.seq, self.starts, self.slots, self.positions, self.taken, PAGE)
        ops.rotary(self.q_turned, self.k_turned, self.q, self.key, self.positions, self.f, self.scale)
        ops.kv8_write(self.k_turned, self.value, self.k, self.v, self.ks, self.vs, self.table, self.seq, self.starts, longest)
        args = self.out, self.lse, self.q_turned, self.k, self.v, self.ks, self.vs, self.table, self.seq
        if longest == 1:
            ops.kv8_decode_attention(*args, D ** -0.5, self.ws)
        else:
            ops.kv8_attention(*args, self.starts, longest, D ** -0.5, self.ws)

    def drop_taken(self):
        self.free = self.free[int(self.taken):].contiguous()

    def check(self, rows_per_request):
        torch.cuda.synchronize()
        assert capi.load_library().device_status() == 0
        seq, starts = self.seq.tolist(), self.starts.tolist()
        T = starts[-1]
        want = reference(self.q_turned[:T], self.k, self.v, self.ks, self.vs, self.table.cpu(), seq, starts, D ** -0.5,
                         tall=rows_per_request * HQ // HKV >= 33 and rows_per_request > 1)
        check(self.out[:T], self.lse[:T], want)


def test_prompts_then_tokens():
    lens, free_pages = [70, 5, 33, 1], 8
    layer = Layer(4, sum(lens) + 3, free_pages)
    layer.feed([0] * 4, lens)
    layer.step(max(lens))
    layer.check(max(lens))
    layer.drop_taken()
    written = [(layer.k_turned[s:e].clone(), layer.value[s:e].clone()) for s, e in zip(layer.starts.tolist(), layer.starts.tolist()[1:])]
    # the reader brings back what was written, to a step of e4m3 (2^-4 of a value, or 2^-10 of a scale, which is below 2^-7 of the largest)
    rows = [torch.zeros((sum(lens), HKV, D), device="cuda") for _ in range(2)]
    ops.kv8_read(*rows, layer.k, layer.v, layer.ks, layer.vs, layer.table, _i32([0] * 4), layer.starts, max(lens))
    for got, i in zip(rows, (0, 1)):
        want = torch.cat([w[i] for w in written]).float()
        assert bool(((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -17 * want.abs().max()).all())
    one = Layer.__new__(Layer)
    one.__dict__.update(layer.__dict__)
    for name in ("q", "key", "value", "q_turned", "k_turned", "out", "lse"):
        setattr(one, name, getattr(layer, name)[:4].clone())
    one.slots, one.positions = layer.slots[:4].clone(), layer.positions[:4].clone()
    for i in range(40):
        one.feed([n + i for n in lens], [1] * 4)
        one.step(1)
        one.drop_taken()
        if i % 13 == 0 or i == 39:
            one.check(1)


def test_captured_steps_follow_the_lengths_of_the_replay():
    layer = Layer(6, 6, 40, seed=1)
    layer.feed([0] * 6, [1] * 6)
    layer.step(1)
    torch.cuda.synchronize()
    # a cache of some length, written by hand; every request has its own pages
    layer.table.copy_(torch.arange(6 * 40, device="cuda", dtype=torch.int32).view(6, 40))
    layer.k.copy_((torch.randn(layer.k.shape, generator=layer.gen, device="cuda") * 100).clamp(-448, 448))
    layer.v.copy_((torch.randn(layer.v.shape, generator=layer.gen, device="cuda") * 100).clamp(-448, 448))
    layer.ks.fill_(2.0 ** -7)
    layer.vs.fill_(2.0 ** -7)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(1)
    for context in ([5, 100, 0, 1000, 31, 32], [1200, 3, 700, 16, 15, 0], [0] * 6):
        layer.feed(context, [1] * 6)
        # (tables and positions: pages that the requests have are kept, new ones come off the list; here all are there already)
        graph.replay()
        torch.cuda.synchronize()
        keep = layer.out.clone(), layer.lse.clone()
        layer.check(1)
        graph.replay()   # the same step again: the same bits
        torch.cuda.synchronize()
        assert torch.equal(layer.out, keep[0]) and torch.equal(layer.lse, keep[1])


def test_a_captured_chunk():
    layer = Layer(3, 90, 20, seed=2)
    layer.feed([0, 0, 0], [60, 20, 10])
    layer.step(60)
    layer.check(60)
    layer.drop_taken()
    free = layer.free.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(60)
    layer.feed([60, 20, 10], [50, 0, 40])
    graph.replay()
    layer.check(60)
    assert torch.equal(layer.free, free)


def test_streams_with_their_own_workspaces():
    """Two layers on two streams, interleaved, against each by itself; and tensors used on a stream other than the one that made them."""
    layers, want = [], []
    for seed in (3, 4):
        layer = Layer(8, 8, 30, seed=seed)
        layer.table.copy_(torch.arange(8 * 30, device="cuda", dtype=torch.int32).view(8, 30))
        layer.k.copy_((torch.randn(layer.k.shape, generator=layer.gen, device="cuda") * 100).clamp(-448, 448))
        layer.v.copy_((torch.randn(layer.v.shape, generator=layer.gen, device="cuda") * 100).clamp(-448, 448))
        layer.ks.fill_(2.0 ** -7)
        layer.vs.fill_(2.0 ** -7)
        layer.feed([100 * seed + 50 * i for i in range(8)], [1] * 8)
        layer.step(1)
        torch.cuda.synchronize()
        layers.append(layer)
        want.append(layer.out.clone())
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(20):
        for layer, stream in zip(layers, streams):
            with torch.cuda.stream(stream):
                layer.out.zero_()
                layer.step(1)
    torch.cuda.synchronize()
    for layer, w in zip(layers, want):
        assert torch.equal(layer.out, w)


def test_calls_behind_one_another_without_a_wait():
    """Each call changes what the one in front of it still reads or writes."""
    layer = Layer(5, 5, 12, seed=5)
    outs = []
    for rounds in range(2):
        layer.free = torch.arange(layer.blocks, dtype=torch.int32, device="cuda")
        layer.gen.manual_seed(9)
        got = []
        context = [0] * 5
        for i in range(30):
            layer.feed(context, [1] * 5)
            layer.step(1)
            # (pages are taken from the list's start by every step that begins one: the same number for all requests)
            if i % PAGE == 0:
                layer.free = layer.free[5:].contiguous()
            context = [c + 1 for c in context]
            got.append(layer.out.clone())
            if rounds == 1:
                torch.cuda.synchronize()
        outs.append(torch.stack(got))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])


def test_nothing_is_allocated_or_synchronised():
    layer = Layer(4, 4, 8, seed=6)
    layer.feed([0] * 4, [1] * 4)
    layer.step(1)
    layer.step(4)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.set_sync_debug_mode("error")
    try:
        layer.step(1)
        layer.step(4)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.cuda.memory_allocated() == before
    torch.cuda.synchronize()
