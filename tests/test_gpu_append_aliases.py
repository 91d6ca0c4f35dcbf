"""The append's result in memory of its inputs: anywhere but q itself it goes
through a copy, so no row is overwritten before it is read."""
import pytest
import torch

from myvllm_amd import paged_kv_append
from myvllm_amd.full_attention import _crosses

BF = torch.bfloat16


def test_what_crosses():
    packed = torch.zeros(9, 12, 64, dtype=BF)
    q, k, v = packed.split([4, 4, 4], 1)
    one = q[:1]
    assert not _crosses(q, q, k, v) and not _crosses(packed[:, :4], q, k, v)
    assert not _crosses(torch.zeros(9, 4, 64, dtype=BF), q, k, v)
    assert _crosses(k, q, k, v) and _crosses(v, q, k, v) and _crosses(packed[:, 1:5], q, k, v)
    assert _crosses(q[1:], q[:-1], k[1:], v[1:])
    assert _crosses(q.transpose(0, 1)[:, :4], q[:4], k, v)  # q's address, another order of rows
    assert _crosses(k, torch.zeros(9, 4, 64, dtype=BF), k, v)
    # in one allocation, apart: one after the other, column blocks of one matrix
    arena = torch.zeros(9 * 4 * 64 * 4, dtype=BF)
    parts = [t.view(9, 4, 64) for t in arena.chunk(4)]
    wide = torch.zeros(9, 16, 64, dtype=BF).split([4, 4, 4, 4], 1)
    for o, *qkv in (parts, wide, wide[::-1], parts[::-1]):
        assert not _crosses(o, *qkv)
    late = torch.zeros(10, 16, 64, dtype=BF)  # the next row's column block
    assert not _crosses(late[1:, 12:], late[:-1, :4], late[:-1, 4:8], late[:-1, 8:12])
    assert _crosses(late[1:, 10:14], late[:-1, :4], late[:-1, 4:8], late[:-1, 8:12])
    # refused by the entry, not copied over
    assert not _crosses(packed, q, k, v) and not _crosses(one, q, k, v)
    assert not _crosses(k.view(torch.float16), q, k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 2000])
def test_out_in_an_input(dev, T):
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(T, 2, 128, generator=g).to(BF).to(dev) for _ in range(3))
    cos, sin = torch.rand(T, 64, generator=g).to(dev), torch.rand(T, 64, generator=g).to(dev)
    pages = -(-T // 16)
    tab = torch.randperm(pages, generator=g).to(torch.int32)[None].to(dev)
    ctx, cu = torch.tensor([T], device=dev), torch.tensor([0, T], device=dev)
    print(f"append into its inputs T={T}", flush=True)

    def run(q, k, v, out=None):
        kc, vc = (torch.zeros(pages, 16, 2, 128, dtype=BF, device=dev) for _ in range(2))
        return paged_kv_append(q, k, v, kc, vc, tab, ctx, 16, cos, sin, cu_seqlens=cu, out=out), kc, vc

    want = run(q, k, v)
    for place in ("k", "v", "next row", "row before", "row order"):
        kk, vv = k.clone(), v.clone()
        if place == "row order":  # from the first row's memory on, in another order
            qq = q.transpose(0, 1).contiguous().transpose(0, 1)
            out = qq.transpose(0, 1).reshape(T, 2, 128)
        else:
            buf = torch.zeros(T + 1, 2, 128, dtype=BF, device=dev)
            qq = buf[1:] if place == "row before" else buf[:-1]
            qq.copy_(q)
            out = {"k": kk, "v": vv, "next row": buf[1:], "row before": buf[:-1]}[place]
        got = run(qq, kk, vv, out)
        assert got[0] is out
        assert all(torch.equal(a, b) for a, b in zip(got, want)), place
