"""GPU tests of attention over the 8-bit paged cache: one-token decode, and any number of tokens under a causal mask, a window or none.

Against the formula in 64 bits, element by element within a bound that follows from the roundings
(``kv8_util.reference``).  Everything that no token of a request sees is NaN: slots behind its end, pages and scales it does not hold.
"""
import math

import pytest
import torch

from pth_flash_attn_b200 import capi, kv8, ops
from tests.kv8_util import E4M3, check, make_cache, make_table, reference

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def workspace(D):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return torch.zeros(kv8.workspace_bytes(D=D, num_sms=sms), dtype=torch.uint8, device="cuda")


class Batch:
    """Requests of ``q_lens`` tokens whose caches hold ``kv_lens``, the tokens among them; what none of them sees is NaN."""

    def __init__(self, kv_lens, q_lens, Hq, Hkv, D, dtype=BF16, *, page=32, group=16, layout="NHD", pad=0, seed=0, spare=3, scale_up=1.0,
                 scales=(-8, -5), foreign=False):
        gen = torch.Generator().manual_seed(seed)
        self.kv_lens, self.D, self.page = list(kv_lens), D, page
        blocks = sum(-(-n // page) for n in kv_lens) + spare
        self.table = make_table(self.kv_lens, page, blocks, gen=gen)
        self.k, self.v, self.ks, self.vs = make_cache(blocks, page, group, Hkv, D, layout, pad=pad)
        cg = torch.Generator(device="cuda").manual_seed(seed)
        for r, n in enumerate(self.kv_lens):
            at = torch.arange(n, device="cuda")
            b, slot = self.table[r].cuda().long()[at // page], at % page
            for cells, scale in ((self.k, self.ks), (self.v, self.vs)):
                cells[b, slot] = (torch.randn((n, Hkv, D), generator=cg, device="cuda") * 100).clamp(-448, 448).to(E4M3)
                s = torch.exp2(torch.randint(*scales, scale.shape, generator=cg, device="cuda").float())
                if foreign:   # (scales of another writer: any positive number)
                    s = s * (1 + torch.rand(scale.shape, generator=cg, device="cuda"))
                scale[b, slot // group] = s[b, slot // group]
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
        self.ws = workspace(D)

    def decode(self, window=0):
        ops.kv8_decode_attention(self.out, self.lse, self.q, self.k, self.v, self.ks, self.vs, self.bt, self.lens, self.D ** -0.5, self.ws, window)
        return self

    def attend(self, window=0, causal=True):
        ops.kv8_attention(self.out, self.lse, self.q, self.k, self.v, self.ks, self.vs, self.bt, self.lens, self.qsl, self.longest_q, self.D ** -0.5,
                          self.ws, window, causal)
        return self

    def check(self, window=0, causal=True, what=""):
        torch.cuda.synchronize()
        assert capi.load_library().device_status() == 0
        check(self.out, self.lse, self.reference(window, causal), what)

    def reference(self, window=0, causal=True):
        rows = self.longest_q * (self.q.shape[1] // self.k.shape[2])
        tall = self.longest_q > 1 and rows >= (17 if self.D == 64 else 33)   # (the rule of kv8_api.cu)
        return reference(self.q, self.k, self.v, self.ks, self.vs, self.table, self.kv_lens, self.starts, self.D ** -0.5, window, causal, tall)


EDGES = [0, 1, 15, 16, 17, 127, 128, 129, 255, 300, 0, 1000]


def _decode(kv_lens, *args, window=0, **kw):
    Batch(kv_lens, [1] * len(kv_lens), *args, **kw).decode(window).check(window)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 8, 64), (12, 2, 256), (16, 1, 128), (32, 2, 64), (40, 2, 256), (64, 1, 128)])
def test_decode_lengths(Hq, Hkv, D, dtype):
    _decode(EDGES, Hq, Hkv, D, dtype, seed=D + Hq)


@pytest.mark.parametrize("page,group", [(16, 16), (32, 32), (48, 16), (48, 48), (64, 16), (816, 48), (816, 816), (128, 64), (80, 80)])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_decode_pages(page, group, layout):
    _decode([2000, 33, 816, 817, 1, 700], 8, 2, 128, BF16, page=page, group=group, layout=layout, pad=16 if page == 48 else 0, seed=page)


@pytest.mark.parametrize("window", [1, 2, 31, 128, 129, 500, 5000])
def test_decode_windows(window):
    _decode([1, 2, 130, 700, 1999, 0], 8, 2, 128, window=window, seed=window)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_pieces_and_heads(D):
    _decode([9000, 20000, 5], 12, 3, D, seed=D)


def test_decode_many_requests():
    lens = [(37 * i * i + 11 * i) % 400 for i in range(700)]
    _decode(lens, 4, 2, 64, seed=5)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("foreign", [False, True])
def test_scales_that_differ(foreign, dtype):
    """Scales over a range of 2^20, later and earlier ones the largest, and scales that are no powers of two."""
    _decode([3000, 400, 129, 17], 8, 2, 128, dtype, scales=(-14, 7), foreign=foreign, seed=9, scale_up=2.0 ** -6)


@pytest.mark.parametrize("size", [-100, -30, 30, 90])
def test_scales_of_any_size(size):
    """Values of 2^size: weights take their unit from the scales, so nothing under- or overflows that the output does not."""
    b = Batch([300, 129, 1000], [1] * 3, 8, 2, 128, scales=(-7, -6), seed=4)
    b.vs.mul_(2.0 ** size)
    b.decode().check()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_large_probability_beside_many_small_ones(dtype):
    """A key with most of the weight in front of keys whose small weights add up: none of them is lost."""
    n, D = 30000, 128
    b = Batch([n], [1], 4, 1, D, dtype, seed=3, scales=(-7, -6))
    at = torch.arange(n, device="cuda")
    where = b.table[0].cuda().long()[at // 32], at % 32
    k = torch.zeros((n, 1, D), device="cuda")
    k[0, 0, 0] = 448.0
    b.k[where] = k.to(E4M3)
    b.q.zero_()
    b.q[:, :, 0] = 11.5 * D ** 0.5 / (448.0 / 128)   # e^-11.5 of the first for every other key, 0.3 of it together
    b.v[where] = (torch.rand((n, 1, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 400 + 40).to(E4M3)
    b.decode().check()


def test_a_later_maximum_moves_the_bound():
    """Scores that grow along the keys, by more than the bound's slack at a time."""
    n, D = 4000, 128
    b = Batch([n], [1], 8, 2, D, seed=3, scales=(-7, -6))
    at = torch.arange(n, device="cuda")
    where = b.table[0].cuda().long()[at // 32], at % 32
    k = torch.zeros((n, 2, D), device="cuda")
    k[..., 0] = (at.float() / n * 440)[:, None]
    b.k[where] = k.to(E4M3)
    b.q.zero_()
    b.q[..., 0] = 200.0
    b.decode().check()


@pytest.mark.parametrize("scale_up", [2.0 ** -60, 2.0 ** -8, 2.0 ** 6])
def test_query_sizes(scale_up):
    b = Batch([500, 64], [1, 1], 8, 2, 128, BF16, scale_up=scale_up, seed=2)
    b.q[0, 1] *= 2.0 ** -20   # (rows of their own size)
    b.decode().check()


def test_bad_blocks_stand_for_zeros_and_the_table_ends_requests():
    b = Batch([200, 300, 128], [1] * 3, 8, 2, 128, seed=6)   # (128: the pages it has are full, so their NaN is not seen)
    b.table[0, 1], b.table[1, 0], b.table[2, 2] = -1, 1 << 20, 77777
    b.bt = b.table.cuda()
    b.kv_lens[2] = 5000   # past the row of the table
    b.lens[2] = 5000
    b.table[2, 4:], b.bt[2, 4:] = -1, -1
    b.decode().check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (16, 16, 64), (12, 2, 256), (64, 2, 128)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 40), (False, 0), (False, 130)])
def test_few_tokens(Hq, Hkv, D, dtype, causal, window):
    """Verification: several tokens of each request, fewer keys than tokens among them."""
    kv, q = [1, 4, 130, 700, 0, 2, 1500, 128, 129], [1, 4, 3, 4, 2, 4, 2, 4, 0]
    Batch(kv, q, Hq, Hkv, D, dtype, seed=D + Hq).attend(window, causal).check(window, causal)


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 4, 64), (12, 2, 256)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 100), (False, 0)])
def test_prompts(Hq, Hkv, D, causal, window):
    kv, q = [300, 37, 1, 900, 128, 500], [300, 37, 1, 130, 100, 0]
    Batch(kv, q, Hq, Hkv, D, seed=D).attend(window, causal).check(window, causal)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D,page,group,layout", [(32, 8, 128, 64, 16, "NHD"), (8, 1, 128, 16, 16, "HND"), (16, 16, 64, 48, 48, "NHD"),
                                                        (6, 1, 256, 816, 48, "HND"), (5, 5, 128, 80, 80, "NHD")])
def test_long_prompts(Hq, Hkv, D, page, group, layout, dtype):
    """Row tiles that several CTAs share, ragged, over pages of every kind."""
    Batch([2300, 700, 64, 1], [500, 700, 1, 1], Hq, Hkv, D, dtype, page=page, group=group, layout=layout, seed=page, pad=16 if page == 48 else 0).attend().check()


@pytest.mark.parametrize("foreign", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompts_over_scales_that_differ(D, foreign):
    Batch([1000, 300], [200, 300], 8, 2, D, scales=(-14, 1), foreign=foreign, seed=7, scale_up=2.0 ** -3).attend().check()


@pytest.mark.parametrize("size", [-100, -30, 30, 90])
def test_prompts_over_scales_of_any_size(size):
    b = Batch([300, 129], [100, 129], 8, 2, 128, scales=(-7, -6), seed=4)
    b.vs.mul_(2.0 ** size)
    b.attend().check()


def test_prompts_of_rows_of_their_own_size():
    b = Batch([500, 64], [100, 64], 8, 2, 128, seed=2)
    b.q[10, 1] *= 2.0 ** -20
    b.q[11, 2] *= 2.0 ** 8
    b.q[12, 3] = 0.0
    b.attend().check()


def test_prompts_with_a_later_maximum():
    n, D = 2000, 128
    b = Batch([n], [120], 4, 1, D, seed=3, scales=(-7, -6))
    at = torch.arange(n, device="cuda")
    k = torch.zeros((n, 1, D), device="cuda")
    k[..., 0] = (at.float() / n * 440)[:, None]
    b.k[b.table[0].cuda().long()[at // 32], at % 32] = k.to(E4M3)
    b.q.zero_()
    b.q[..., 0] = 200.0
    b.attend().check()


def test_prompts_over_bad_blocks_and_past_the_table():
    b = Batch([400, 300, 256], [100, 300, 200], 8, 2, 128, seed=6)
    b.table[0, 1], b.table[1, 2], b.table[2, 7] = -1, 1 << 20, 77777
    b.bt = b.table.cuda()
    # tokens whose own positions are past the row of the table: they see what there is
    b.kv_lens[2] = b.table.shape[1] * 32 + 50
    b.lens[2] = b.kv_lens[2]
    b.table[2, 8:], b.bt[2, 8:] = -1, -1
    b.attend().check()


def test_more_tokens_than_keys():
    """Lengths below the number of tokens: the first of them are at negative positions and see nothing."""
    b = Batch([40, 3, 0], [60, 5, 4], 8, 2, 128, seed=1)
    b.attend().check()
    Batch([40, 3, 0], [4, 4, 4], 8, 2, 128, seed=1).attend().check()
    Batch([2, 1, 0], [4, 4, 4], 8, 2, 128, seed=1).attend().check()


def test_one_token_through_both_calls():
    """A single token's call and a call of one token each give the same."""
    b = Batch(EDGES, [1] * len(EDGES), 8, 2, 128, seed=1)
    first = b.decode(50).out.clone(), b.lse.clone()
    b.out.fill_(math.nan)
    b.attend(50).check(50)
    assert torch.equal(first[0], b.out) and torch.equal(first[1], b.lse)


def test_tokens_past_the_bound_and_behind_the_last_request_are_left():
    b = Batch([200, 100], [5, 3], 8, 2, 128, seed=8)
    whole = b.attend().out.clone()
    b.out.fill_(7.0)
    b.lse.fill_(7.0)
    b.longest_q = 3
    b.qsl[2] = 7   # one token of the second request less: a padding row
    b.kv_lens[1] = 99
    b.lens[1] = 99
    b.attend()
    torch.cuda.synchronize()
    assert torch.equal(b.out[:3], whole[:3]) and bool((b.out[3:5] == 7).all()) and bool((b.out[7:] == 7).all()) and bool((b.lse[7:] == 7).all())
    assert not bool((b.out[5:7] == 7).any())


def test_nothing_to_do():
    b = Batch([0, 0], [1, 1], 8, 2, 64, seed=0)
    b.decode().check()
    e = Batch([], [], 8, 2, 64)
    e.decode()
    e.attend()
    z = Batch([50], [0], 8, 2, 64)
    z.attend()
    torch.cuda.synchronize()


def test_without_lse():
    b = Batch([300], [1], 8, 2, 128, seed=2)
    want = b.decode().out.clone()
    b.out.fill_(0)
    b.lse = torch.empty(0, device="cuda")
    b.decode()
    assert torch.equal(b.out, want)


def test_a_workspace_serves_calls_of_any_shape_and_the_bits_repeat():
    ws = workspace(128)
    batches = [Batch([9000, 100], [1, 1], 8, 2, 128, seed=1), Batch([40, 3000, 2, 900], [4] * 4, 8, 2, 128, seed=2),
               Batch([20000], [1], 64, 2, 128, F16, seed=3), Batch([700, 2000], [200, 50], 8, 2, 128, seed=4)]
    want = []
    for rounds in range(3):
        for i, b in enumerate(batches):
            b.ws = ws
            b.out.fill_(math.nan)
            b.decode() if b.longest_q == 1 else b.attend()
            if rounds == 0:
                b.check()
                want.append((b.out.clone(), b.lse.clone()))
            else:
                assert torch.equal(b.out, want[i][0]) and torch.equal(b.lse, want[i][1])
    assert not bool(ws[:4096].any()), "arrival counters are left at zero"


def test_a_small_workspace_is_refused():
    b = Batch([300], [1], 8, 2, 128)
    b.ws = b.ws[:1 << 16]
    with pytest.raises(RuntimeError, match="kv8_decode_attention: workspace has 65536 bytes"):
        b.decode()


def test_offsets_past_32_bits():
    """Cells and scales more than 2^31 bytes and elements from the first."""
    page, Hkv, D = 16, 1, 64
    blocks = (2 ** 31 + 2 ** 27) // (page * D)
    cells = torch.full((blocks, page, Hkv, D), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
    store = torch.full((1 << 12,), math.nan, device="cuda")
    scale = store.as_strided((blocks, 1, Hkv), (0, 1, 1))
    scale.fill_(1.0 / 128)
    b = Batch([100, 50], [1, 1], 4, 1, D, page=16, seed=1)
    b.table = torch.tensor([[blocks - 1 - 3 * i for i in range(7)], [blocks // 2 + i for i in range(7)]], dtype=torch.int32)
    b.bt = b.table.cuda()
    gen = torch.Generator(device="cuda").manual_seed(3)
    for r, n in enumerate(b.kv_lens):
        at = torch.arange(n, device="cuda")
        cells[b.bt[r].long()[at // page], at % page] = (torch.randn((n, Hkv, D), generator=gen, device="cuda") * 100).clamp(-448, 448).to(E4M3)
    b.k = b.v = cells
    b.ks = b.vs = scale
    b.decode().check()


def _sees(b, r, i, key, window, causal):
    """Whether token i of request r sees a key."""
    own = b.kv_lens[r] - (b.starts[r + 1] - b.starts[r]) + i
    return (not causal or key <= own) and (not window or key > own - window) and key < b.kv_lens[r]


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 8, 64), (12, 2, 256), (16, 2, 128)])
@pytest.mark.parametrize("kv,q", [([300, 4, 140], [4, 3, 2]), ([700, 300, 90], [260, 300, 33])])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 70), (False, 50)])
def test_nan_under_keys_that_some_tokens_do_not_see(Hq, Hkv, D, kv, q, causal, window):
    """NaN among the keys and values of a request's own tokens: it reaches the tokens that see it, in a value only its dimension,
    and no other.  (Values: their weight of zero times NaN would be NaN.)"""
    b = Batch(kv, q, Hq, Hkv, D, seed=D, spare=0)
    clean = b.reference(window, causal)
    want_out, want_lse = (x.clone() for x in clean[:2])
    gen = torch.Generator().manual_seed(1)
    G = Hq // Hkv
    for r, (n, t) in enumerate(zip(kv, q)):
        for key in {n - 1, n - t // 2 - 1, max(0, n - t - 3), max(0, n - window), int(torch.randint(n, (1,), generator=gen))}:
            h, d = int(torch.randint(Hkv, (1,), generator=gen)), int(torch.randint(D, (1,), generator=gen))
            block, slot = int(b.table[r, key // b.page]), key % b.page
            b.v[block, slot, h, d] = math.nan
            for i in range(t):
                if _sees(b, r, i, key, window, causal):
                    want_out[b.starts[r] + i, h * G:(h + 1) * G, d] = math.nan
        key, h = n - 1 - t // 3, int(torch.randint(Hkv, (1,), generator=gen))
        b.k[int(b.table[r, key // b.page]), key % b.page, h, 3] = math.nan
        for i in range(t):
            if _sees(b, r, i, key, window, causal):
                want_out[b.starts[r] + i, h * G:(h + 1) * G] = math.nan
                want_lse[b.starts[r] + i, h * G:(h + 1) * G] = math.nan
    b.attend(window, causal)
    torch.cuda.synchronize()
    assert capi.load_library().device_status() == 0
    assert torch.equal(b.out.isnan(), want_out.isnan()) and torch.equal(b.lse.isnan(), want_lse.isnan())
    ok = ~want_out.isnan()
    assert bool(((b.out.double() - clean[0]).abs() <= clean[2])[ok].all())


def test_nan_among_the_keys_that_all_tokens_see():
    """NaN far from the tokens' own keys, where nothing is masked; and for a single token."""
    for q in ([1, 1], [4, 4], [200, 1]):
        b = Batch([900, 500], q, 8, 2, 128, seed=3)
        block, slot = int(b.table[0, 100 // b.page]), 100 % b.page
        b.v[block, slot, 1, 7] = math.nan
        b.attend() if max(q) > 1 else b.decode()
        nan = torch.zeros_like(b.out, dtype=torch.bool)
        nan[:q[0], 4:8, 7] = True
        assert torch.equal(b.out.isnan(), nan)


@pytest.mark.parametrize("q_lens", [[1, 1], [4, 3], [200, 130]])
def test_scales_that_are_broadcast(q_lens):
    """One scale for a whole cache: strides of zero."""
    b = Batch([300, 140], q_lens, 8, 2, 128, seed=8)
    b.ks, b.vs = (torch.full((1, 1, 1), s, device="cuda").expand(b.ks.shape) for s in (2.0 ** -7, 0.013))
    b.attend().check()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_scale_that_is_no_number_reaches_the_rows_that_see_it(D):
    """Prompts over keys, and values, of which a block's scale is NaN: NaN where a row sees the block, the others as they are."""
    for which in ("ks", "vs"):
        b = Batch([200, 90], [200, 60], 16, 2, D, seed=D)
        page, slot = divmod(100, b.page)
        scales = getattr(b, which)
        was = scales.clone()
        scales[int(b.table[0][page]), slot // 16] = math.nan
        b.attend()
        torch.cuda.synchronize()
        assert capi.load_library().device_status() == 0
        first = 100 // 16 * 16
        assert bool(b.out[first:200].isnan().all()) and bool(b.out[:first].isfinite().all()) and bool(b.out[200:].isfinite().all())
        setattr(b, which, was)
        want = b.reference()
        keep = torch.cat([torch.arange(first), torch.arange(200, 260)]).cuda()
        check(b.out[keep], b.lse[keep], tuple(x[keep] for x in want))


def test_scales_of_minus_zero():
    """Values of a scale of -0 are zeros, and take nothing from the blocks behind them."""
    b = Batch([400, 90], [300, 60], 16, 2, 128, seed=2)
    b.vs[b.table[0].cuda().long()[:4]] = -0.0
    b.attend().check()
