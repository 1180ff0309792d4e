"""An `out` that shares memory with what the call reads is refused: workgroups write while others still read."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)


def test_out_of_a_read_out_over_its_inputs(rt):
    r = rt.Readout4.quantize(torch.ones((1, 64, 2, 32), device="cuda"))
    mem = torch.zeros(4 * 64 + 64, device="cuda")
    x = mem[:4 * 64].view(4, 64)
    bits = mem[:8].view(torch.int32).view(4, 2)
    live = mem[100:101].view(torch.int32)
    live.fill_(32)
    for call in (lambda: r.matvec(x, out=x.view(4, 2, 32)),
                 lambda: r.matvec(x, out=mem[63:63 + 256].view(4, 2, 32)),
                 lambda: r.matvec(x, out=r.records.view(-1)[64:64 + 1024].view(torch.float32).view(4, 2, 32)),
                 lambda: r.logits(bits, out=mem[7:7 + 256].view(4, 2, 32)),
                 lambda: r.probabilities(bits.clone(), live, out=mem[:256].view(4, 2, 32))):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    # side by side, and where the rows have to be copied first
    want = r.matvec(x)
    assert torch.equal(r.matvec(x, out=torch.empty((4, 2, 32), device="cuda")), want)
    wide = torch.randn((4, 128), device="cuda")
    first = wide[:, ::2].contiguous()
    assert torch.equal(r.matvec(wide[:, ::2], out=wide.view(-1)[:256].view(4, 2, 32)), r.matvec(first))
    out = torch.empty(4 * 64 + 8, device="cuda")
    out[:8].view(torch.int32).zero_()
    assert torch.all(r.logits(out[:8].view(torch.int32).view(4, 2), out=out[8:].view(4, 2, 32)) == 0)
