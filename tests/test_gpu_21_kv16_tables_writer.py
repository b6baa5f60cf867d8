"""GPU tests of the 16-bit cache's writer (bit for bit) and of the tables made from request lengths (whole numbers)."""
import numpy as np
import pytest
import torch

from pth_flash_attn_b200 import ops
from tests.kv16_util import make_cache, tables_reference

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("src", [F32, BF16, F16])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,Hkv,page,layout,pad", [(64, 1, 16, "NHD", 0), (128, 3, 5, "HND", 8), (256, 2, 24, "NHD", 16), (128, 8, 1, "NHD", 0)])
def test_writer_rounds_and_places_every_row(D, Hkv, page, layout, pad, dtype, src):
    gen = torch.Generator(device="cuda").manual_seed(D + page)
    blocks, T = 40, min(37, 40 * page - 3)
    k, v = make_cache(blocks, page, Hkv, D, dtype, layout, pad=pad, gen=gen)
    whole = k._base if k._base is not None else k
    want_storage = whole.clone()
    slots = torch.randperm(blocks * page, generator=gen, device="cuda")[:T]
    slots[[1, T - 1]] = torch.tensor([-1, -7], device="cuda")     # padding
    slots[3] = blocks * page                                      # outside the cache
    wide = torch.randn((2, T, Hkv + 1, D + 8), generator=gen, device="cuda").to(src)
    for key, value in ((wide[0, :, :Hkv, :D], wide[1, :, 1:, 8:]),                              # strided, on 16-byte boundaries
                       (wide[0, :, :Hkv, 1:D + 1], wide[1, :, :Hkv, 3:D + 3]),                  # on none
                       (wide[0, :, :Hkv, :D].contiguous(), wide[1, :, :1, :D].expand(T, Hkv, D))):   # heads that share a row
        whole.copy_(want_storage)
        ek, ev = k.clone(), v.clone()
        live = (slots >= 0) & (slots < blocks * page)
        b, s = slots[live] // page, slots[live] % page
        ek[b, s], ev[b, s] = key[live].float().to(dtype), value[live].float().to(dtype)
        ops.kv16_write(key, value, k, v, slots)
        torch.cuda.synchronize()
        assert torch.equal(k.view(torch.int16), ek.view(torch.int16)) and torch.equal(v.view(torch.int16), ev.view(torch.int16))
        if pad:
            assert torch.equal(whole[..., D:], want_storage[..., D:])


@pytest.mark.parametrize("src", [F32, BF16, F16])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_writer_special_values(dtype, src):
    x = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), 1e-8, -1e-8, 65504.0, 65520.0, 3.4e38, 1.00390625, 1.01171875] * 6, device="cuda")[:64]
    key = x.to(src).view(1, 1, 64)
    k, v = make_cache(1, 16, 1, 64, dtype, fill=1.0)
    ops.kv16_write(key, -key, k, v, torch.tensor([5], device="cuda"))
    torch.cuda.synchronize()
    for got, want in ((k[0, 5, 0], key[0, 0].float().to(dtype)), (v[0, 5, 0], (-key)[0, 0].float().to(dtype))):
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(got[~nan].view(torch.int16), want[~nan].view(torch.int16))


def test_writer_offsets_past_32_bits():
    Hkv, D, page = 8, 128, 16
    blocks = (5 << 30) // (page * Hkv * D * 2)
    k = torch.empty((blocks, page, Hkv, D), dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    key, value = torch.randn((2, 3, Hkv, D), device="cuda").to(BF16)
    slots = torch.tensor([blocks * page - 1, 0, (blocks - 7) * page + 3], device="cuda")
    ops.kv16_write(key, value, k, v, slots)
    torch.cuda.synchronize()
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(k[s // page, s % page], key[i]) and torch.equal(v[s // page, s % page], value[i])


def test_writer_no_tokens():
    k, v = make_cache(2, 16, 2, 64, BF16, fill=1.0)
    none = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    ops.kv16_write(none, none, k, v, torch.empty(0, dtype=torch.int64, device="cuda"))
    torch.cuda.synchronize()
    assert bool((k == 1).all())


def _tables(context, new, num_free, width, num_tokens, block_size, *, seed=0, extra_rows=0):
    rng = np.random.default_rng(seed)
    R = len(context)
    ids = rng.permutation(1 << 20)
    table = ids[:R * width].reshape(R, width).astype(np.int32) if R * width <= 1 << 19 else rng.integers(0, 1 << 20, (R, width), dtype=np.int32)
    free = ids[-num_free:].astype(np.int32) if num_free else np.zeros(0, np.int32)
    want = tables_reference(context, new, free.tolist(), table, num_tokens, block_size)
    i32 = dict(dtype=torch.int32, device="cuda")
    bt = torch.full((R + extra_rows, width + 3), -9, **i32)[:, :width]      # rows of a wider table
    bt[:R] = torch.from_numpy(table).cuda()
    seq, starts = torch.full((R,), -9, **i32), torch.full((R + 1,), -9, **i32)
    slots, positions = (torch.full((num_tokens,), -9, dtype=torch.int64, device="cuda") for _ in range(2))
    taken = torch.full((1,), -9, **i32)
    ops.page_tables(torch.tensor(context, **i32), torch.tensor(new, **i32), torch.from_numpy(free).cuda(), bt, seq, starts, slots, positions,
                    taken, block_size)
    torch.cuda.synchronize()
    for got, expected, name in ((bt[:R], want[0], "block_table"), (seq, want[1], "seq_lens"), (starts, want[2], "query_start_loc"),
                                (slots, want[3], "slot_mapping"), (positions, want[4], "positions"), (taken, [want[5]], "pages_taken")):
        assert got.tolist() == [list(x) if isinstance(x, list) else x for x in expected], name
    if extra_rows:
        assert bool((bt[R:] == -9).all())
    assert bool((bt._base[:, width:] == -9).all())


@pytest.mark.parametrize("block_size", [1, 5, 16, 64, 816])
@pytest.mark.parametrize("R,longest_q,longest_c", [(1, 1, 0), (3, 40, 100), (64, 1, 3000), (17, 700, 1000), (300, 9, 50)])
def test_tables(R, longest_q, longest_c, block_size):
    rng = np.random.default_rng(R + block_size)
    new, context = rng.integers(0, longest_q + 1, R).tolist(), rng.integers(0, longest_c + 1, R).tolist()
    width = -(-(longest_q + longest_c) // block_size)
    pages = sum(-(-(c + q) // block_size) - -(-c // block_size) for c, q in zip(context, new))
    _tables(context, new, pages + 5, width, sum(new) + 3, block_size, seed=R, extra_rows=2)


def test_tables_page_edges():
    _tables([0, 15, 16, 17, 31, 32, 0, 5], [16, 1, 1, 15, 2, 0, 0, 11], 20, 4, 46, 16)


def test_tables_of_requests_without_anything():
    _tables([0, 0, 0], [0, 0, 0], 2, 1, 2, 16)
    _tables([], [], 2, 1, 3, 16)
    _tables([-3, 4], [2, -5], 3, 2, 4, 4)


def test_tables_free_list_too_short():
    """The pages past the list are -1, their tokens have no slot, and pages_taken says how many were needed."""
    _tables([10, 0, 30, 5], [30, 100, 1, 50], 6, 12, 190, 16)
    _tables([10, 0], [30, 100], 0, 12, 130, 16)


def test_tables_rows_too_short():
    _tables([10, 0, 60], [100, 20, 30], 40, 4, 150, 16)


def test_tables_more_tokens_than_the_arrays_hold():
    _tables([10, 0, 60], [100, 20, 30], 40, 8, 77, 16)


@pytest.mark.parametrize("R", [255, 256, 257, 1000, 5000, 16384])
def test_tables_many_requests(R):
    rng = np.random.default_rng(R)
    _tables(rng.integers(0, 60, R).tolist(), rng.integers(0, 5, R).tolist(), 8 * R, 4, 5 * R, 16, seed=R)


def test_tables_one_long_request():
    _tables([100000, 3], [100000, 1], 7000, 12600, 100001, 16)


def test_tables_without_positions():
    i32 = dict(dtype=torch.int32, device="cuda")
    bt, slots = torch.zeros((2, 4), **i32), torch.zeros(5, dtype=torch.int64, device="cuda")
    ops.page_tables(torch.tensor([3, 0], **i32), torch.tensor([2, 3], **i32), torch.tensor([7, 8, 9], **i32), bt, torch.zeros(2, **i32),
                    torch.zeros(3, **i32), slots, torch.empty(0, dtype=torch.int64, device="cuda"), torch.zeros(1, **i32), 4)
    # request 0 goes on in its page 0 (slot 3), then takes page 7; request 1 takes page 8
    assert slots.tolist() == [3, 28, 32, 33, 34] and bt.tolist() == [[0, 7, 0, 0], [8, 0, 0, 0]]


def test_tables_graph_replay():
    i32 = dict(dtype=torch.int32, device="cuda")
    context, new = torch.tensor([3, 0], **i32), torch.tensor([2, 3], **i32)
    args = (context, new, torch.tensor([7, 8, 9], **i32), torch.zeros((2, 4), **i32), torch.zeros(2, **i32), torch.zeros(3, **i32),
            torch.zeros(5, dtype=torch.int64, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda"), torch.zeros(1, **i32), 4)
    ops.page_tables(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.page_tables(*args)
    context.copy_(torch.tensor([0, 4]))
    new.copy_(torch.tensor([1, 1]))
    args[3].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert args[6].tolist() == [28, 32, -1, -1, -1] and args[3].tolist() == [[7, 0, 0, 0], [0, 8, 0, 0]] and args[8].item() == 2
