"""One layer of an encoder-decoder model, served from a 16-bit paged cache, with the operators of ``ops``:

    python examples/encoder_decoder_step.py            # needs a B200

A batch of requests arrives with documents of every length (their encoder states) and prompts of every length:

1. ``page_tables`` gives the documents pages and slots, ``kv16_write`` stores the encoder's keys and values there;
2. the prompts' tokens look at the documents with ``kv16_cross_attention``, and get pages of the self-attention cache;
3. tokens are generated one by one: ``page_tables`` moves every request on by one token, ``kv16_write`` stores its key and
   value, ``kv16_decode_attention`` attends over what the request has said, ``kv16_cross_attention`` over its document.
   The step is captured in a CUDA graph once and replayed: lengths, pages and slots live on the GPU.

Every result is compared with torch in 64 bits.
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from pth_flash_attn_b200 import kv16, ops  # noqa: E402

HQ, HKV, D, PAGE, STEPS = 16, 4, 64, 16, 6
DTYPE = torch.bfloat16


class PagedCache:
    """A layer's 16-bit cache with its free pages, and the tables that ``page_tables`` keeps up to date."""

    def __init__(self, num_reqs, max_len, num_tokens, device):
        i32 = dict(dtype=torch.int32, device=device)
        pages = -(-max_len // PAGE)
        self.k, self.v = torch.full((2, num_reqs * pages, PAGE, HKV, D), float("nan"), dtype=DTYPE, device=device)
        self.free = torch.randperm(num_reqs * pages, device=device).to(torch.int32)
        self.block_table = torch.zeros((num_reqs, pages), **i32)
        self.lens = torch.zeros(num_reqs, **i32)
        self.seq_lens = torch.zeros(num_reqs, **i32)
        self.starts = torch.zeros(num_reqs + 1, **i32)
        self.slots = torch.zeros(num_tokens, dtype=torch.int64, device=device)
        self.positions = torch.zeros(num_tokens, dtype=torch.int64, device=device)
        self.taken = torch.zeros(1, **i32)

    def extend(self, new_lens, key, value):
        """Gives every request pages for its new tokens and stores their keys and values."""
        n = key.shape[0]
        ops.page_tables(self.lens, new_lens, self.free, self.block_table, self.seq_lens, self.starts, self.slots[:n],
                        self.positions[:n], self.taken, PAGE)
        ops.kv16_write(key, value, self.k, self.v, self.slots[:n])
        self.lens.copy_(self.seq_lens)
        # (the pages that were taken leave the front of the list; its length stays what the captured call has, and the pool has
        # pages for every request's longest, so none of them comes round to the front again)
        at = (torch.arange(len(self.free), device=key.device) + self.taken) % len(self.free)
        self.free.copy_(self.free[at])


def attention_in_64_bits(q, keys, values):
    """q [t, HQ, D] over keys / values [n, HKV, D]."""
    rows = q.double().view(len(q), HKV, HQ // HKV, D)
    scores = torch.einsum("thgd,jhd->thgj", rows, keys.double()) * D ** -0.5
    return torch.einsum("thgj,jhd->thgd", torch.softmax(scores, -1), values.double()).reshape(q.shape)


def check(name, out, want):
    error = float((out.double() - want).norm() / want.norm())
    print(f"{name:>28}: relative error {error:.1e}")
    assert error < 5e-3, name


def main():
    device = torch.device("cuda")
    torch.manual_seed(0)
    document_lens, prompt_lens = [700, 33, 1500, 129, 1], [40, 300, 7, 1, 64]
    R = len(document_lens)
    i32 = dict(dtype=torch.int32, device=device)

    def normal(*shape):
        return torch.randn(shape, device=device).to(DTYPE)

    workspace = torch.zeros(kv16.workspace_bytes(D=D, num_sms=torch.cuda.get_device_properties(device).multi_processor_count),
                            dtype=torch.uint8, device=device)
    no_lse = torch.empty(0, device=device)

    # the documents
    documents = PagedCache(R, max(document_lens), sum(document_lens), device)
    ek, ev = normal(sum(document_lens), HKV, D), normal(sum(document_lens), HKV, D)
    documents.extend(torch.tensor(document_lens, **i32), ek, ev)
    per_document = list(zip(ek.split(document_lens), ev.split(document_lens)))

    # the prompts: cross attention of many tokens, and the start of the self-attention cache
    said = PagedCache(R, max(prompt_lens) + STEPS, sum(prompt_lens), device)
    pk, pv, pq = (normal(sum(prompt_lens), h, D) for h in (HKV, HKV, HQ))
    said.extend(torch.tensor(prompt_lens, **i32), pk, pv)
    history = [[k, v] for k, v in zip(pk.split(prompt_lens), pv.split(prompt_lens))]
    out = torch.empty_like(pq)
    ops.kv16_cross_attention(out, no_lse, pq, documents.k, documents.v, documents.block_table, documents.seq_lens, said.starts,
                             max(prompt_lens), D ** -0.5, workspace)
    check("prompts over documents", out, torch.cat([attention_in_64_bits(q, *kv) for q, kv in zip(pq.split(prompt_lens), per_document)]))

    # the generated tokens: one captured step, replayed
    one = torch.ones(R, **i32)
    key, value, q = (torch.zeros((R, h, D), dtype=DTYPE, device=device) for h in (HKV, HKV, HQ))
    self_out, cross_out = torch.empty_like(q), torch.empty_like(q)

    def step():
        said.extend(one, key, value)
        ops.kv16_decode_attention(self_out, no_lse, q, said.k, said.v, said.block_table, said.seq_lens, D ** -0.5, workspace)
        ops.kv16_cross_attention(cross_out, no_lse, q, documents.k, documents.v, documents.block_table, documents.seq_lens,
                                 said.starts, 1, D ** -0.5, workspace)

    def new_token():
        for x in (key, value, q):
            x.copy_(torch.randn_like(x))
        for r in range(R):
            history[r] = [torch.cat([history[r][0], key[r:r + 1]]), torch.cat([history[r][1], value[r:r + 1]])]

    graph = None
    for i in range(STEPS):
        new_token()
        if graph is None:
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):   # (captures, does not run)
                step()
        else:
            graph.replay()
        check(f"token {i}, over what was said", self_out, torch.cat([attention_in_64_bits(q[r:r + 1], *history[r]) for r in range(R)]))
        check(f"token {i}, over documents", cross_out, torch.cat([attention_in_64_bits(q[r:r + 1], *per_document[r]) for r in range(R)]))
    assert said.seq_lens.tolist() == [n + STEPS for n in prompt_lens]


if __name__ == "__main__":
    main()
