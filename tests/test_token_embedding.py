"""Embedding lookup with scaling and the gradient of its table by sorted tokens:
refusals on the CPU, values and gradients against 64 bits on the GPU."""
import pytest
import torch

from metallora_b200 import _lib, kernels, ops
from metallora_b200.exceptions import ConfigurationError, DeviceError, ShapeError
from metallora_b200.layers import LoRAEmbedding, TokenEmbedding

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def test_refusals():
    table, idx = torch.zeros(10, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(DeviceError):
        ops.embedding(idx, table)
    for pad in (10, -11):
        with pytest.raises(ConfigurationError):
            ops.embedding(idx, table, padding_idx=pad)
    with pytest.raises(ShapeError):
        ops.embedding(idx, table[0])
    for kw in ({"num_embeddings": 0}, {"embedding_dim": 0}, {"padding_idx": 5}):
        with pytest.raises(ConfigurationError):
            TokenEmbedding(**{"num_embeddings": 5, "embedding_dim": 8, **kw})
    assert TokenEmbedding(5, 8, padding_idx=-1).padding_idx == 4
    lib, p = _lib.load(), 1 << 20
    for kw in ({"T": 0}, {"V": 0}, {"D": 0}, {"dtype": 3}, {"idx": None}, {"idx": p + 4}, {"x": p + 1},
               {"T": 1 << 31}):
        v = {"idx": p, "x": p, "T": 4, "V": 10, "D": 8, "dtype": 0, **kw}
        assert lib.mlora_embedding_forward(v["idx"], v["x"], p, v["T"], v["V"], v["D"], 1.0,
                                           v["dtype"], None) < 0, kw
        assert lib.mlora_embedding_backward(v["idx"], v["x"], p, v["T"], v["V"], v["D"], 1.0, -1,
                                            v["dtype"], p, 1 << 30, None) < 0, kw
    assert lib.mlora_embedding_backward(p, p, p, 4, 10, 8, 1.0, -1, 0, p, 16, None) == \
        _lib.MLORA_ERR_WORKSPACE
    assert lib.mlora_embedding_backward(p, p, p, 4, 10, 8, 1.0, -1, 0, p + 8, 1 << 30, None) == \
        _lib.MLORA_ERR_WORKSPACE


def _check(idx, table, dy, scale=1.0, padding_idx=None):
    dtype = table.dtype
    h = torch.finfo(dtype).eps / 2
    sub = 2.0 ** -25 if dtype == FP16 else 0.0
    table.requires_grad_(True)
    out = ops.embedding(idx, table, scale=scale, padding_idx=padding_idx)
    assert out.shape == (*idx.shape, table.shape[1]) and out.dtype == dtype
    flat = idx.reshape(-1).long()
    rows = table.detach().double()[flat] * scale
    e = (out.detach().double().reshape(rows.shape) - rows).abs()
    assert (e <= 1.01 * h * rows.abs() + 2.0 ** -23 * rows.abs() + sub).all()
    grad = torch.autograd.grad(out, table, dy)[0]
    d = dy.double().reshape(rows.shape)
    if padding_idx is not None:
        d = d * (flat != padding_idx % table.shape[0])[:, None]
    want = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
    sums = want.clone().index_add_(0, flat, d.abs()) * abs(scale)
    want.index_add_(0, flat, d).mul_(scale)
    count = torch.bincount(flat, minlength=table.shape[0])[:, None]
    # n sums in 32 bits and the scaling, then one rounding
    bound = 1.01 * h * want.abs() + (count + 2) * 2.0 ** -24 * sums + sub
    assert ((grad.double() - want).abs() <= bound).all()
    assert torch.count_nonzero(grad[count[:, 0] == 0]) == 0
    again = kernels.embedding_bwd(dy, idx, table.shape[0], scale,
                                  None if padding_idx is None else padding_idx % table.shape[0])
    assert torch.equal(grad, again)
    assert _lib.device_status(reset=True) == 0


def _case(t, v, d, dtype, seed=0, hot=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    idx = torch.randint(0, v, (t,), generator=g, device="cuda")
    if hot:
        idx[torch.rand(t, generator=g, device="cuda") < hot] = v // 2
    return (idx, torch.randn((v, d), generator=g, device="cuda").to(dtype),
            torch.randn((t, d), generator=g, device="cuda").to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("t,v,d", [(1, 1, 1), (1, 50, 8), (31, 3, 33), (32, 1, 64), (33, 1, 100),
                                   (64, 9, 24), (65, 2, 24), (300, 40, 1001), (512, 100, 40), (513, 100, 40),
                                   (2048, 500, 72), (2049, 500, 8), (5000, 70000, 264),
                                   (9000, 30, 520), (16384, 9000, 16), (20001, 3000, 24)])
def test_values_and_gradients(cuda, dtype, t, v, d):
    idx, table, dy = _case(t, v, d, dtype, seed=t)
    _check(idx, table, dy, scale=1.7)


@pytest.mark.gpu
@pytest.mark.parametrize("hot", [0.3, 1.0])
@pytest.mark.parametrize("t", [100, 4500])
def test_common_and_padding_entries(cuda, t, hot):
    """Runs that cross many chunks; the padding entry has no gradient."""
    idx, table, dy = _case(t, 64, 136, FP32, seed=t, hot=hot)
    _check(idx, table, dy)
    _check(idx, table, dy, scale=0.5, padding_idx=32)
    _check(idx, table, dy, padding_idx=-1)


@pytest.mark.gpu
def test_sums_in_token_order(cuda):
    """A run's sum is that of its tokens in order wherever the chunks' borders cut it:
    small whole numbers, which fp32 adds exactly, and a large one that cancels."""
    idx, table, _ = _case(1000, 7, 16, FP32, seed=2)
    dy = torch.randint(-50, 50, (1000, 16), device=cuda).float()
    grad = kernels.embedding_bwd(dy, idx, 7)
    want = torch.zeros(7, 16, device=cuda, dtype=torch.float64).index_add_(0, idx, dy.double())
    assert torch.equal(grad.double(), want)


@pytest.mark.gpu
def test_indices_outside_the_table(cuda):
    idx, table, dy = _case(40, 30, 64, BF16)
    bad = idx.clone()
    bad[3], bad[4], bad[39] = 30, -1, (1 << 32) + 2  # the last would be 2 in 32 bits
    _lib.device_status(reset=True)
    out = kernels.embedding_fwd(bad, table)
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == 0x107
    grad = kernels.embedding_bwd(dy, bad, 30)
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == 0x107
    off = torch.zeros(40, dtype=torch.bool, device=cuda)
    off[[3, 4, 39]] = True
    assert torch.count_nonzero(out[off]) == 0 and torch.equal(out[~off], table[idx[~off]])
    zero = dy.masked_fill(off[:, None], 0)
    assert torch.equal(grad, kernels.embedding_bwd(zero, idx, 30))


@pytest.mark.gpu
def test_shapes_strides_and_empty_batches(cuda):
    idx, table, dy = _case(60, 20, 24, BF16, seed=4)
    want = ops.embedding(idx, table)
    got = ops.embedding(idx.reshape(3, 20).int(), table.t().contiguous().t())
    assert got.shape == (3, 20, 24) and torch.equal(got.reshape(60, 24), want)
    assert torch.equal(ops.embedding(idx.reshape(20, 3).t(), table), table[idx.reshape(20, 3).t()])
    table.requires_grad_(True)
    flat = torch.zeros(table.numel() + 1, dtype=BF16, device=cuda)[1:].view(20, 24)  # 2 bytes off
    flat.copy_(table.detach())
    assert torch.equal(ops.embedding(idx, flat), want)
    ones = torch.ones((), dtype=BF16, device=cuda).expand(60, 24)  # a broadcast gradient
    g = torch.autograd.grad(ops.embedding(idx, table), table, ones)[0]
    assert torch.equal(g.double(), torch.bincount(idx, minlength=20).double()[:, None].expand(20, 24))
    e = ops.embedding(idx[:0], table)
    assert e.shape == (0, 24)
    assert torch.count_nonzero(torch.autograd.grad(e.sum(), table)[0]) == 0


@pytest.mark.gpu
def test_graph_and_streams(cuda):
    idx, table, dy = _case(3000, 200, 64, BF16, seed=5)
    table.requires_grad_(True)
    static = idx.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.embedding(static, table, scale=2.0)
        grad = torch.autograd.grad(out, table, dy)[0]
    static.copy_(idx.flip(0))
    graph.replay()
    want = ops.embedding(static, table, scale=2.0)
    gw = torch.autograd.grad(want, table, dy)[0]
    assert torch.equal(out, want) and torch.equal(grad, gw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w2 = ops.embedding(static, table, scale=2.0)
        g2 = torch.autograd.grad(w2, table, dy)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(w2, want) and torch.equal(g2, gw)


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    idx, table, dy = _case(500, 40, 32, FP32, seed=6)
    grad = kernels.embedding_bwd(dy, idx, 40, scale=1.5)
    step = torch.randn_like(table)

    def f(t):
        return (ops.embedding(idx, t, scale=1.5).double() * dy.double()).sum()
    slope = float(f(table + step) - f(table - step)) / 2  # linear: no higher terms
    assert abs(slope - float((grad.double() * step.double()).sum())) < 1e-4 * float(dy.abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_lora_embedding_with_a_trained_base(cuda, dtype):
    emb = LoRAEmbedding(300, 128, rank=8, freeze_base=False, device=cuda, dtype=dtype)
    with torch.no_grad():
        emb.B.normal_(0, 0.1)
    idx = torch.randint(0, 300, (4, 50), device=cuda)
    dy = torch.randn(4, 50, 128, device=cuda).to(dtype)
    emb(idx).backward(dy)
    assert torch.equal(emb.embeddings.grad, kernels.embedding_bwd(dy, idx, 300))
    da, db = kernels.lora_embedding_bwd(dy, idx, emb.A, emb.B, emb.alpha)
    assert torch.equal(emb.A.grad, da.to(dtype)) and torch.equal(emb.B.grad, db.to(dtype))
    emb.A.requires_grad_(False)
    emb.B.requires_grad_(False)
    emb.zero_grad()
    emb(idx).backward(dy)  # of the table alone
    assert emb.A.grad is None and torch.equal(emb.embeddings.grad, kernels.embedding_bwd(dy, idx, 300))


@pytest.mark.gpu
def test_module_and_a_head_that_shares_the_table(cuda):
    emb = TokenEmbedding(500, 64, scale=8.0, padding_idx=0, device=cuda, dtype=BF16)
    idx = torch.randint(0, 500, (3, 40), device=cuda)
    idx[:, 30:] = 0
    hidden = emb(idx)
    labels = idx.clone()
    labels[idx == 0] = -100
    loss = ops.linear_cross_entropy(hidden, emb.weight, labels)
    loss.backward()
    both = emb.weight.grad
    h = hidden.detach().requires_grad_(True)
    w = emb.weight.detach().clone().requires_grad_(True)
    dh, dw = torch.autograd.grad(ops.linear_cross_entropy(h, w, labels), (h, w))
    de = kernels.embedding_bwd(dh, idx, 500, 8.0, 0)
    assert torch.equal(both, de + dw)
    assert torch.count_nonzero(de[0]) == 0 and torch.count_nonzero(dw[0]) > 0


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    v, d = 530_000, 4096
    table = torch.zeros(v, d, device=cuda, dtype=FP16)
    idx = torch.tensor([0, v - 1, 7, v - 1, v - 2], device=cuda)
    table[idx] = torch.randn(5, d, device=cuda).to(FP16)
    assert torch.equal(ops.embedding(idx, table), table[idx])
    dy = torch.randn(5, d, device=cuda).to(FP16)
    grad = kernels.embedding_bwd(dy, idx, v)
    assert torch.equal(grad[v - 2], dy[4]) and torch.equal(grad[7], dy[2])
    assert torch.equal(grad[v - 1], (dy[1].float() + dy[3].float()).to(FP16))
    assert torch.count_nonzero(grad[8:v - 2]) == 0



@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_at_every_offset(cuda, dtype):
    """Rows that begin and end anywhere in 16 bytes, the table's first and last among them;
    a scale of two is exact."""
    for d in (*range(1, 20), 31, 33, 63, 65, 130, 257, 1001, 2049, 4097):
        for start in (0, 1, 3, 7):
            held = torch.randn(start + 5 * d, device=cuda).to(dtype)
            table = held[start:].view(5, d)
            idx = torch.tensor([4, 0, 2, 4, 1, 3, 0], device=cuda)
            assert torch.equal(kernels.embedding_fwd(idx, table, 2.0), table[idx] * 2)
    _lib.device_status(reset=True)
    idx = torch.tensor([4, 9, 0, -1], device=cuda)  # two of no row of this table
    out = kernels.embedding_fwd(idx, table, 2.0)
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == 0x107
    assert torch.equal(out[::2], table[[4, 0]] * 2) and not out[1::2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 15, 16, 17, 32, 33, 48, 63, 64, 65, 80, 512, 513])
def test_runs_across_chunks(cuda, t):
    """Runs that begin, end and go on at every border; fp32 sums of at most t terms are off
    by (t - 1) additions, the scale and the store: under (t + 1) half steps of the
    terms' magnitudes."""
    g = torch.Generator(device="cuda").manual_seed(t)
    for v, d in ((1, 36), (2, 37), (5, 600), (40, 512), (1000, 1030)):
        dy = torch.randn(t, d, device=cuda, generator=g)
        idx = torch.randint(0, v, (t,), device=cuda, generator=g)
        padding = 0 if v == 5 else None
        grad = kernels.embedding_bwd(dy, idx, v, 3.0, padding)
        terms = dy.double() if padding is None else dy.double() * (idx != padding)[:, None]
        want, size = (torch.zeros(v, d, device=cuda, dtype=torch.float64).index_add_(0, idx, 3 * x)
                      for x in (terms, terms.abs()))
        assert ((grad.double() - want).abs() <= (t + 1) * torch.finfo(torch.float32).eps / 2 * size).all()
        assert torch.equal(grad, kernels.embedding_bwd(dy, idx, v, 3.0, padding))
