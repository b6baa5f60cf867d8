"""GPU tests of attention over the 16-bit paged cache: one-token decode and cross attention.

Against the formula in 64 bits, element by element within a bound that follows from the roundings
(``kv16_util.reference``).  Everything that a request does not see is NaN: slots behind its end, pages it does not hold.
"""
import math

import pytest
import torch

from pth_flash_attn_b200 import capi, kv16, ops
from tests.kv16_util import check, make_cache, make_table, reference

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _workspace(D):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return torch.zeros(max(256, kv16.workspace_bytes(D=D, num_sms=sms)), dtype=torch.uint8, device="cuda")


class Batch:
    """Requests of ``q_lens`` tokens over ``kv_lens`` keys; what none of them sees is NaN."""

    def __init__(self, kv_lens, q_lens, Hq, Hkv, D, dtype, *, page=16, layout="NHD", pad=0, seed=0, spare=3, scale_up=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.kv_lens, self.D, self.Hq, self.page = list(kv_lens), D, Hq, page
        blocks = sum(-(-n // page) for n in kv_lens) + spare
        self.table = make_table(self.kv_lens, page, blocks, gen=gen)
        self.k, self.v = make_cache(blocks, page, Hkv, D, dtype, layout, pad=pad, fill=math.nan)
        cg = torch.Generator(device="cuda").manual_seed(seed)
        for r, n in enumerate(self.kv_lens):
            at = torch.arange(n, device="cuda")
            where = self.table[r].cuda().long()[at // page], at % page
            self.k[where] = torch.randn((n, Hkv, D), generator=cg, device="cuda").to(dtype)
            self.v[where] = torch.randn((n, Hkv, D), generator=cg, device="cuda").to(dtype)
        self.starts = [0]
        for n in q_lens:
            self.starts.append(self.starts[-1] + n)
        T = self.starts[-1]
        # (rows of a wider tensor: strides that are not the sizes')
        self.q = (torch.randn((T, Hq + 1, D), generator=cg, device="cuda") * scale_up).to(dtype)[:, :Hq]
        self.out = torch.full((T, Hq + 2, D), math.nan, dtype=dtype, device="cuda")[:, 1:Hq + 1]
        self.lse = torch.full((T, Hq), math.nan, device="cuda")
        self.lens = torch.tensor(self.kv_lens, dtype=torch.int32, device="cuda")
        self.qsl = torch.tensor(self.starts, dtype=torch.int32, device="cuda")
        self.longest_q = max(q_lens, default=0)
        self.bt = self.table.cuda()
        self.ws = _workspace(D)

    def decode(self, window=0):
        ops.kv16_decode_attention(self.out, self.lse, self.q, self.k, self.v, self.bt, self.lens, self.D ** -0.5, self.ws, window)
        return self

    def cross(self):
        ops.kv16_cross_attention(self.out, self.lse, self.q, self.k, self.v, self.bt, self.lens, self.qsl, self.longest_q,
                                 self.D ** -0.5, self.ws)
        return self

    def check(self, window=0, what=""):
        torch.cuda.synchronize()
        assert capi.load_library().device_status() == 0
        check(self.out, self.lse, reference(self.q, self.k, self.v, self.table, self.kv_lens, self.starts, self.D ** -0.5, window), what)


EDGES = [0, 1, 15, 16, 17, 127, 128, 129, 255, 300, 0, 1000]


def _decode(kv_lens, *args, window=0, **kw):
    Batch(kv_lens, [1] * len(kv_lens), *args, **kw).decode(window).check(window)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 2, 128), (6, 1, 256), (16, 16, 64), (3, 3, 128), (20, 2, 128), (32, 2, 64),
                                      (32, 2, 256), (66, 2, 128), (64, 1, 64), (64, 1, 256), (12, 4, 256)])
def test_decode_heads_and_types(Hq, Hkv, D, dtype):
    _decode(EDGES, Hq, Hkv, D, dtype, seed=Hq + D)


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 100, 816])
@pytest.mark.parametrize("pad", [0, 8])
def test_decode_pages_and_strides(page, layout, pad):
    _decode(EDGES + [2000], 8, 2, 128, BF16, page=page, layout=layout, pad=pad, seed=page)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 129, 200, 999, 1000, 5000, 1 << 31])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_window(window, D):
    _decode(EDGES, 8, 2, D, BF16, window=window, seed=window % 1000)


@pytest.mark.parametrize("kv_lens", [[1], [2], [40000], [0], [0, 0, 0], [131], [9000, 3], [1] * 700, list(range(0, 900, 3)), [5, 20000, 0, 130, 7000]])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 1, 128), (32, 8, 128), (4, 4, 64), (12, 2, 256)])
def test_decode_lengths(kv_lens, Hq, Hkv, D):
    _decode(kv_lens, Hq, Hkv, D, BF16, seed=len(kv_lens))


def test_decode_more_heads_than_multiprocessors():
    _decode([300, 0, 129, 1000], 400, 400, 64, BF16, seed=2)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decode_large_scores(dtype):
    """Scores of +-100: the running maximum moves far, and one key holds nearly all of a row's weight."""
    _decode([700, 128, 1, 3000], 8, 2, 128, dtype, scale_up=30.0, seed=5)


@pytest.mark.parametrize("step", [0.25, -0.25])
def test_decode_scores_that_rise_or_fall(step):
    """The largest score sits in the last (first) tile, by a margin that grows tile by tile."""
    b = Batch([2000, 40], [1, 1], 8, 2, 128, BF16, seed=6)
    b.q.fill_(1.0)
    at = torch.arange(2000, device="cuda")
    b.k[b.table[0].cuda().long()[at // 16], at % 16] = (at * step / 128 * 11.3)[:, None, None].to(BF16).expand(-1, 2, 128)
    b.decode().check()


def test_decode_probabilities_of_equal_keys():
    """All keys alike: every probability is 1 / n, whatever their number."""
    b = Batch([1, 128, 129, 5000], [1] * 4, 8, 2, 128, F16, seed=7)
    for r, n in enumerate(b.kv_lens):
        at = torch.arange(n, device="cuda")
        b.k[b.table[r].cuda().long()[at // 16], at % 16] = 0.5
    b.decode().check()


def test_decode_infinite_score_follows_the_formula():
    """An infinite query makes its row NaN, as in the formula, and no other."""
    b = Batch([300, 300], [1, 1], 8, 2, 128, BF16, seed=8)
    b.q[0, 3] = math.inf
    b.decode()
    torch.cuda.synchronize()
    assert bool(torch.isnan(b.out[0, 3]).all())
    keep = torch.ones(2, 8, dtype=torch.bool, device="cuda")
    keep[0, 3] = False
    q = b.q.clone()
    q[0, 3] = 0
    want = reference(q, b.k, b.v, b.table, b.kv_lens, b.starts, 128 ** -0.5)
    check(b.out[keep][None], b.lse[keep][None], [w[keep][None] for w in want])


def test_decode_without_lse():
    b = Batch(EDGES, [1] * len(EDGES), 8, 2, 128, BF16, seed=9)
    lse, b.lse = b.lse, torch.empty(0, device="cuda")
    b.decode()
    b.lse = lse
    other = Batch(EDGES, [1] * len(EDGES), 8, 2, 128, BF16, seed=9).decode()
    torch.cuda.synchronize()
    assert torch.equal(b.out, other.out) and bool(torch.isnan(lse).all())


def test_decode_writes_nothing_else():
    b = Batch(EDGES, [1] * len(EDGES), 8, 2, 128, BF16, seed=10)
    wide = b.out._base if b.out._base is not None else b.out
    b.decode()
    torch.cuda.synchronize()
    assert bool(torch.isnan(wide[:, 0]).all()) and bool(torch.isnan(wide[:, -1]).all())


def test_decode_offsets_past_32_bits():
    """A cache of 5 GB whose used pages lie at its end."""
    Hkv, D, page, kv_lens = 8, 128, 16, [500, 77, 2000]
    blocks = (5 << 30) // (page * Hkv * D * 2)
    storage = torch.empty((2, blocks, page, Hkv, D), dtype=BF16, device="cuda")
    pages = [-(-n // page) for n in kv_lens]
    table = torch.zeros((3, max(pages)), dtype=torch.int32)
    last = blocks
    for r, n in enumerate(pages):
        table[r, :n] = torch.arange(last - n, last, dtype=torch.int32)
        last -= n
    storage[:, last:].normal_()
    q = torch.randn((3, 32, D), device="cuda").to(BF16)
    out, lse = torch.empty_like(q), torch.empty((3, 32), device="cuda")
    ops.kv16_decode_attention(out, lse, q, storage[0], storage[1], table.cuda(), torch.tensor(kv_lens, dtype=torch.int32, device="cuda"),
                              D ** -0.5, _workspace(D))
    check(out, lse, reference(q, storage[0], storage[1], table, kv_lens, [0, 1, 2, 3], D ** -0.5))


def test_decode_shared_pages():
    """Requests that share a prefix share its pages."""
    b = Batch([512, 300, 640], [1] * 3, 8, 2, 128, BF16, seed=11)
    b.table[1, :16] = b.table[0, :16]
    b.table[2, :16] = b.table[0, :16]
    b.bt = b.table.cuda()
    b.decode().check()


Q_LENS = [1, 0, 2, 7, 64, 1, 130, 300, 5, 0, 33, 256]
STATES = [40, 9, 0, 128, 500, 129, 1000, 77, 1, 0, 2000, 256]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 2, 128), (6, 1, 256), (4, 4, 64), (2, 2, 128), (10, 2, 128), (64, 1, 64), (33, 1, 256),
                                      (16, 2, 256)])
def test_cross_heads_and_types(Hq, Hkv, D, dtype):
    Batch(STATES, Q_LENS, Hq, Hkv, D, dtype, seed=Hq + D).cross().check()


@pytest.mark.parametrize("q_lens", [[1] * 12, [2] * 12, [0, 1] * 6, [3, 1, 2, 0] * 3, [4] * 12, [9] * 12, [16] * 12, [40] * 12, [128] * 12])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 4, 64), (12, 2, 256)])
def test_cross_short_queries(q_lens, Hq, Hkv, D):
    Batch(STATES, q_lens, Hq, Hkv, D, BF16, seed=sum(q_lens)).cross().check()


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 816])
@pytest.mark.parametrize("pad", [0, 8])
def test_cross_pages_and_strides(page, layout, pad):
    Batch(STATES, Q_LENS, 4, 2, 128, BF16, page=page, layout=layout, pad=pad, seed=page).cross().check()


@pytest.mark.parametrize("q_lens,states", [([1], [1]), ([1000], [1]), ([1], [30000]), ([600], [30000]), ([257], [129]), ([2048, 1], [3, 2048]),
                                           ([1] * 600, list(range(600))), ([31] * 90, list(range(0, 900, 10)))])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 1, 128), (8, 8, 64), (4, 2, 256)])
def test_cross_lengths(q_lens, states, Hq, Hkv, D):
    Batch(states, q_lens, Hq, Hkv, D, BF16, seed=len(q_lens)).cross().check()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_cross_large_scores(dtype):
    Batch([700, 128, 1, 3000], [70, 200, 130, 257], 8, 2, 128, dtype, scale_up=30.0, seed=5).cross().check()


def test_cross_tokens_past_the_bound_are_left():
    b = Batch([300, 200], [100, 50], 8, 2, 128, BF16, seed=12)
    b.longest_q = 60
    b.cross()
    torch.cuda.synchronize()
    assert bool(torch.isnan(b.out[60:100]).all())
    want = reference(b.q, b.k, b.v, b.table, b.kv_lens, b.starts, 128 ** -0.5)
    kept = torch.cat([torch.arange(60), torch.arange(100, 150)]).cuda()
    check(b.out[kept], b.lse[kept], [w[kept] for w in want])


def test_cross_padding_tokens_are_left():
    """Tokens behind the last request's (a captured batch's padding) keep their content."""
    b = Batch([300, 200], [10, 300], 8, 2, 128, BF16, seed=13)
    b.starts = [0, 10, 250]
    b.qsl = torch.tensor(b.starts, dtype=torch.int32, device="cuda")
    b.longest_q = 300
    b.cross()
    torch.cuda.synchronize()
    assert bool(torch.isnan(b.out[250:]).all())
    want = reference(b.q, b.k, b.v, b.table, b.kv_lens, b.starts, 128 ** -0.5)
    check(b.out[:250], b.lse[:250], [w[:250] for w in want])


@pytest.mark.parametrize("call", ["decode", "cross"])
def test_repeats_are_the_same_bits_and_leave_the_workspace_ready(call):
    kv_lens = [20000, 3, 500, 129, 0, 4000]
    b = Batch(kv_lens, [1] * 6 if call == "decode" else [1, 40, 300, 3, 9, 130], 8, 2, 128, BF16, seed=14)
    getattr(b, call)().check()
    first, flush = b.out.clone(), torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for _ in range(20):
        b.out.fill_(math.nan)
        flush.zero_()
        getattr(b, call)()
        assert torch.equal(b.out, first)


def test_one_workspace_serves_calls_of_every_shape():
    """The same workspace, behind one another, for both calls and for head sizes, groups and lengths of all kinds."""
    ws = max((_workspace(D) for D in (64, 128, 256)), key=len)
    batches = [Batch([9000, 40, 700], q, Hq, Hkv, D, BF16, seed=i)
               for i, (q, Hq, Hkv, D) in enumerate([([1] * 3, 8, 2, 128), ([1, 70, 300], 8, 2, 128), ([1] * 3, 64, 1, 256), ([4, 4, 4], 4, 4, 64),
                                                    ([1] * 3, 3, 1, 64), ([500, 1, 1], 6, 1, 256)])]
    for _ in range(3):
        for b in batches:
            b.ws = ws
            b.decode() if b.starts == [0, 1, 2, 3] else b.cross()
    for b in batches:
        b.check()


@pytest.mark.parametrize("call", ["decode", "cross"])
def test_graph_replay_follows_the_lengths(call):
    """A captured call serves other lengths: nothing of them is baked in."""
    kv_lens = [3000, 10, 500, 1]
    b = Batch(kv_lens, [1] * 4 if call == "decode" else [30, 1, 200, 3], 8, 2, 128, BF16, seed=15)
    getattr(b, call)()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        getattr(b, call)()
    for other in ([3000, 10, 500, 1], [1, 0, 17, 1], [2999, 9, 1, 0]):
        b.kv_lens = other
        b.lens.copy_(torch.tensor(other, dtype=torch.int32))
        b.out.fill_(math.nan)
        graph.replay()
        b.check(what=str(other))


def test_another_stream():
    b = Batch([5000, 40], [1, 1], 8, 2, 128, BF16, seed=16)
    c = Batch([5000, 40], [300, 2], 8, 2, 128, BF16, seed=17)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.decode()
    c.cross()
    torch.cuda.synchronize()
    b.check()
    c.check()


def test_dependent_calls_see_each_other():
    """write -> decode -> a copy of the result, with nothing synchronised in between."""
    b = Batch([4000, 33, 700], [1] * 3, 8, 2, 128, BF16, seed=18)
    key, value = torch.randn((2, 3, 2, 128), device="cuda").to(BF16)
    slots = torch.tensor([int(b.table[r, (n - 1) // 16]) * 16 + (n - 1) % 16 for r, n in enumerate(b.kv_lens)], device="cuda")
    results = []
    for i in range(30):
        ops.kv16_write(key * (i % 3), value, b.k, b.v, slots)
        b.decode()
        results.append(b.out.clone())
        torch.cuda.synchronize() if i < 3 else None
    torch.cuda.synchronize()
    for i in range(30):
        assert torch.equal(results[i], results[i % 3]), i
    b.check()


def test_allocates_nothing_and_does_not_synchronise():
    b, c = Batch([700, 40], [1, 1], 8, 2, 128, BF16), Batch([700, 40], [200, 3], 8, 2, 128, BF16)
    b.decode(), c.cross()
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    torch.cuda.set_sync_debug_mode("error")
    try:
        b.decode(), c.cross()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before


def test_no_requests_and_no_tokens():
    b = Batch([5], [1], 8, 2, 128, BF16)
    empty = torch.empty((0, 8, 128), dtype=BF16, device="cuda")
    ops.kv16_decode_attention(empty, b.lse[:0], empty, b.k, b.v, b.bt[:0], b.lens[:0], 1.0, b.ws)
    ops.kv16_cross_attention(empty, b.lse[:0], empty, b.k, b.v, b.bt, b.lens, b.qsl.zero_(), 0, 1.0, b.ws)
    torch.cuda.synchronize()


def test_refusals_on_the_device():
    b = Batch([40, 50], [1, 1], 8, 2, 128, BF16)
    with pytest.raises(RuntimeError, match="kv16_decode_attention: workspace has 100 bytes"):
        ops.kv16_decode_attention(b.out, b.lse, b.q, b.k, b.v, b.bt, b.lens, 1.0, b.ws[:100])
    with pytest.raises(RuntimeError, match="workspace must be on the same device as q"):
        ops.kv16_decode_attention(b.out, b.lse, b.q, b.k, b.v, b.bt, b.lens, 1.0, b.ws.cpu())
    k = torch.zeros((4, 16, 2, 132), dtype=BF16, device="cuda")[..., 4:]
    with pytest.raises(RuntimeError, match="k_cache.data must be 16-byte aligned"):
        ops.kv16_decode_attention(b.out, b.lse, b.q, k, k, b.bt, b.lens, 1.0, b.ws)
    v = torch.zeros((*b.k.shape[:3], 136), dtype=BF16, device="cuda")[..., :128]
    with pytest.raises(RuntimeError, match="must have the same strides"):
        ops.kv16_cross_attention(b.out, b.lse, b.q, b.k, v, b.bt, b.lens, b.qsl, 1, 1.0, b.ws)


OUTSIDE = [-1, -(1 << 31), 1 << 30, "one past the last"]


@pytest.mark.parametrize("page", [5, 16, 64])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [1, 9, 2, 0], [300, 70, 129, 5]])
def test_block_ids_outside_the_cache_are_keys_of_zeros(q_lens, D, page):
    """Pages that a table does not hold (a free list that ran dry enters -1): no memory behind the cache is read."""
    b = Batch([1000, 300, 129, 40], q_lens, 8, 2, D, BF16, page=page, seed=19)
    zeros = next(i for i in range(b.k.shape[0]) if not bool((b.table == i).any()))
    b.k[zeros], b.v[zeros] = 0, 0
    bad = b.table.clone()
    for r, n in enumerate(b.kv_lens):
        last = -(-n // page) - 1
        for at, block in ((0, OUTSIDE[r % 4]), (last // 2, OUTSIDE[(r + 1) % 4]), (last, OUTSIDE[(r + 2) % 4])):
            bad[r, at] = b.k.shape[0] if isinstance(block, str) else block
            b.table[r, at] = zeros
    b.bt = bad.cuda()
    if max(q_lens) == 1:
        b.decode().check()
    b.cross().check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [300, 70, 129, 5]])
def test_keys_past_the_row_of_the_table_do_not_exist(q_lens, D):
    """A length that the block table has no room for ends where the table does."""
    b = Batch([1000, 300, 960, 40], q_lens, 8, 2, D, BF16, seed=20)
    b.bt = b.bt[:, :60]
    b.kv_lens[0] = 960
    b.lens[2] = (1 << 31) - 1
    if max(q_lens) == 1:
        b.decode().check()
    b.cross().check()


def test_tables_without_columns():
    b = Batch([40, 300], [1, 1], 8, 2, 128, BF16, seed=21)
    b.bt, b.kv_lens = b.bt[:, :0], [0, 0]
    b.decode().check()
    b.cross().check()
