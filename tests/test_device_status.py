"""The device status word: an index outside its table (0x107) loses no arrival.  It
stops and delays no kernel, and a wait that runs out after it is recorded in its place."""
import re
from pathlib import Path

import pytest
import torch

from metallora_b200 import _lib, kernels, ops, quant

CSRC = Path(__file__).resolve().parents[1] / "metallora_b200" / "csrc"
BF16 = torch.bfloat16


def test_one_rule_for_the_word():
    """record_status writes over 0 and, with a wait's code, over an index's; whoever asks
    whether a wait has failed asks wait_failed."""
    ptx = re.sub(r"//[^\n]*", "", (CSRC / "ptx.cuh").read_text())
    body = ptx[ptx.index("void record_status("):]
    body = re.sub(r"\s+", "", body[:body.index("\n}")])
    assert "if(atomicCAS(status,0u,code)==kDevBadIndex&&code!=kDevBadIndex)" \
        "atomicCAS(status,static_cast<uint32_t>(kDevBadIndex),code);" in body
    assert "code!=0&&code!=kDevBadIndex" in re.sub(r"\s+", "", ptx[ptx.index("bool wait_failed("):])
    users = 0
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        assert not re.search(r"\*\s*reinterpret_cast<(const )?volatile uint32_t\*>\((p\.)?status\)", text), path
        users += text.count("wait_failed(")
    assert users == 4  # head_gemm, mx_gemm, tc_gemm, tc_qgemm


@pytest.fixture
def standing(cuda):
    """A call that leaves 0x107, as a function."""
    table = torch.ones(8, 64, device=cuda, dtype=BF16)
    bad = torch.tensor([3, 8], device=cuda)

    def leave():
        _lib.device_status(reset=True)
        ops.embedding(bad, table)
        torch.cuda.synchronize()
        assert _lib.device_status() == 0x107
    yield leave
    _lib.device_status(reset=True)


@pytest.mark.gpu
def test_a_wait_that_runs_out_replaces_an_index(cuda, standing):
    """Rank 0 of a two-rank exchange whose peer never raises its flags gives up after the
    wait budget; an index after it changes nothing."""
    n = 1024
    bufs = [torch.randn(n, device=cuda) for _ in range(2)]
    flags = [torch.zeros(4, dtype=torch.int32, device=cuda) for _ in range(2)]
    counter = torch.zeros(4, dtype=torch.int32, device=cuda)
    pointers = [torch.tensor([t.data_ptr() for t in ts], dtype=torch.int64, device=cuda)
                for ts in (bufs, flags)]
    out = torch.empty_like(bufs[0])
    standing()
    st = _lib.load().mlora_peer_allreduce(
        pointers[0].data_ptr(), pointers[1].data_ptr(), 0, 2, 1, out.data_ptr(), n, 0.5,
        counter.data_ptr(), torch.cuda.current_stream().cuda_stream)
    _lib.check(st, "mlora_peer_allreduce")
    torch.cuda.synchronize()
    assert _lib.device_status() == 0x108
    ops.embedding(torch.tensor([9], device=cuda), torch.ones(8, 64, device=cuda, dtype=BF16))
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == 0x108


def _products(cuda):
    gen = torch.Generator(device=cuda).manual_seed(0)
    x, w, a, b = (torch.randn(*s, device=cuda, generator=gen).to(BF16) * 0.1
                  for s in ((512, 256), (512, 256), (16, 256), (512, 16)))
    out = {"lora": lambda: kernels.lora_linear_fwd(x, w, a, b, 32.0)}
    for name, scheme, group, kw in (("nf4", "nf4", 64, {"lean": True}), ("mxfp4", "mxfp4", None, {})):
        qw = quant.quantize(w, scheme, group, **kw) if group else quant.quantize(w, scheme, **kw)
        out[name] = lambda qw=qw: kernels.qlora_linear_fwd(x, qw, a, b, 32.0)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["lora", "nf4", "mxfp4"])
def test_an_index_delays_no_product(cuda, standing, name):
    """The products' grace time after a failed wait is 200 us a launch, twenty of them 4 ms;
    of these sizes one takes some 10 us."""
    call = _products(cuda)[name]

    def run():
        call()
        torch.cuda.synchronize()
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        for _ in range(20):
            out = call()[0]
        end.record()
        torch.cuda.synchronize()
        return start.elapsed_time(end), out
    _, want = run()
    standing()
    ms, got = run()
    assert _lib.device_status() == 0x107
    assert torch.equal(got, want) and ms < 20 * 0.15
