"""The split decode kernel alone, for every way that lanes share a token: 4 to 32 of
them by head size, type and group."""
import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE = 16


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 128), (8, 8, 128), (16, 8, 64), (32, 8, 256),
                                                  (8, 8, 256), (64, 8, 128), (8, 2, 64)])
def test_split_decode(heads, kv_heads, dim, dtype, cap, monkeypatch):
    import flashinfer_amd as fi
    from flashinfer_amd import decode

    monkeypatch.setattr(decode, "_FUSED_MAX_KV", 0)
    lens = [5, 700, 33, 1, 2049]
    torch.manual_seed(heads + dim)
    pages = [(n + PAGE - 1) // PAGE for n in lens]
    indptr = torch.tensor([0, *torch.tensor(pages).cumsum(0)], dtype=torch.int32, device="cuda")
    order = torch.randperm(sum(pages), device="cuda")
    last = torch.tensor([(n - 1) % PAGE + 1 for n in lens], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(sum(pages), PAGE, kv_heads, dim, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(len(lens), heads, dim, device="cuda").to(dtype)
    w = fi.BatchDecodeWithPagedKVCacheWrapper(
        torch.empty(64 << 20, dtype=torch.uint8, device="cuda"), "NHD", use_tensor_cores=False)
    w.plan(indptr, order.int(), last, heads, kv_heads, dim, PAGE, q_data_type=dtype,
           logits_soft_cap=cap)
    assert not w._fused and not w._tc
    out = w.run(q, (k, v))
    scale = dim ** -0.5
    for i, n in enumerate(lens):
        own = order[indptr[i]:indptr[i + 1]]
        kk, vv = (t[own].flatten(0, 1)[:n].double().repeat_interleave(heads // kv_heads, 1)
                  for t in (k, v))
        qi = q[i].double()
        s = scale * torch.einsum("hd,nhd->hn", qi, kk)
        # a sum of `dim` products and six roundings on the way to the exponent
        off = scale * dim * 2.0 ** -24 * torch.einsum("hd,nhd->hn", qi.abs(), kk.abs()) \
            + 6 * 2.0 ** -24 * s.abs()
        if cap:
            s = cap * torch.tanh(s / cap)
            off = off + 8 * 2.0 ** -24 * cap
        p = torch.softmax(s, -1)
        want = torch.einsum("hn,nhd->hd", p, vv)
        # weights of the softmax off by twice that, and a sum of n of them
        rel = 2 * off.amax(-1, keepdim=True) + (n + 16) * 2.0 ** -24
        bound = rel * torch.einsum("hn,nhd->hd", p, vv.abs())
        bound = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + 2.0 ** -25
        assert ((out[i].double() - want).abs() <= bound).all(), f"request of {n}"
