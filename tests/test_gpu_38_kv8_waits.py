"""GPU tests of the bounded waits of the 8-bit cache's attention kernels: a warp of one CTA stops short, the CTA's waits run out, the kernel ends by
itself and says so, and the next call is as good as ever."""
import pytest
import torch

from pth_flash_attn_b200 import capi
from tests.test_gpu_29_kv8_attention import BF16, Batch

pytestmark = pytest.mark.gpu
STATUS = {"short": 32, "tall": 64}


def _args(b, decode):
    a = capi.new_args(capi.PthB200Kv8Args)
    a.q, a.q_stride_token, a.q_stride_head = b.q.data_ptr(), b.q.stride(0) * 2, b.q.stride(1) * 2
    a.out, a.out_stride_token, a.out_stride_head = b.out.data_ptr(), b.out.stride(0) * 2, b.out.stride(1) * 2
    a.lse = b.lse.data_ptr()
    for s, t in ((a.k_cache, b.k), (a.v_cache, b.v), (a.k_scale, b.ks), (a.v_scale, b.vs)):
        s.data, s.stride_block, s.stride_slot, s.stride_head = t.data_ptr(), *(x * t.element_size() for x in t.stride()[:3])
    a.block_table, a.block_table_row_stride, a.seq_lens = b.bt.data_ptr(), b.bt.stride(0), b.lens.data_ptr()
    a.query_start_loc = None if decode else b.qsl.data_ptr()
    a.workspace, a.workspace_bytes = b.ws.data_ptr(), b.ws.numel()
    a.dtype, a.num_blocks, a.block_size, a.scale_tokens = capi.BF16, b.k.shape[0], b.page, b.page // b.ks.shape[1]
    a.num_kv_heads, a.num_q_heads, a.head_size = b.k.shape[2], b.q.shape[1], b.D
    a.num_reqs, a.num_tokens, a.num_pages = len(b.kv_lens), b.q.shape[0], b.bt.shape[1]
    a.max_query_len, a.causal, a.softmax_scale = b.longest_q, 1, b.D ** -0.5
    return a


def _batch(kernel):
    """Some pieces for every CTA: whole requests, and divided ones."""
    if kernel == "short":
        return Batch([700] * 500 + [60000], [1] * 501, 8, 2, 128, BF16, seed=1)
    return Batch([500] * 60 + [9000], [200] * 60 + [300], 16, 4, 128, BF16, seed=1)


def _run_held(kernel, *what):
    b = _batch(kernel)
    run = b.decode if kernel == "short" else b.attend
    run().check()
    first = b.out.clone()
    lib = capi.load_library()
    assert lib.test_kv8_held(_args(b, kernel == "short"), *what, stream=torch.cuda.current_stream().cuda_stream) == capi.OK, lib.last_error()
    torch.cuda.synchronize()
    assert lib.device_status() == STATUS[kernel]
    assert lib.device_status() == 0   # (read once)
    b.ws.zero_()
    b.out.fill_(float("nan"))
    run().check()
    assert torch.equal(b.out, first)


@pytest.mark.parametrize("after", [0, 1, 2])
@pytest.mark.parametrize("kernel", ["short", "tall"])
def test_schedule_that_stops(kernel, after):
    """Every other warp waits for a piece that does not come."""
    _run_held(kernel, 1, after)


@pytest.mark.parametrize("after", [0, 1, 7, 30])
@pytest.mark.parametrize("kernel", ["short", "tall"])
def test_copies_that_stop(kernel, after):
    """The warp that fills the rings leaves between two units, its boxes in flight."""
    _run_held(kernel, 2, after)


@pytest.mark.parametrize("after", [0, 3])
@pytest.mark.parametrize("kernel", ["short", "tall"])
def test_mmas_that_stop(kernel, after):
    _run_held(kernel, 3, after)


def test_refusals():
    lib = capi.load_library()
    b = Batch([40], [1], 8, 2, 64, BF16)
    assert lib.test_kv8_held(_args(b, True), 1, 0) == capi.EINVAL and "128 dims" in lib.last_error()
    b = Batch([40], [1], 8, 2, 128, BF16)
    for role, after in ((0, 0), (4, 0), (1, -1)):
        assert lib.test_kv8_held(_args(b, True), role, after) == capi.EINVAL and "role must be" in lib.last_error()
