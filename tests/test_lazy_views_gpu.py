"""Tensors whose conjugation or sign is still to be applied: their bytes are not their values."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)


def test_reordered_conjugates(rt):
    p = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    z = torch.tensor([1 + 2j, 3 - 4j], device="cuda")
    with pytest.raises(ValueError, match="alike"):
        rt.beam_reorder([z.conj()], p, out=[torch.empty_like(z)])
    want = z.conj().resolve_conj().flip(0)
    assert torch.equal(rt.beam_reorder([z.conj().resolve_conj()], p, out=[torch.empty_like(z)])[0], want)
    assert torch.equal(rt.beam_reorder([z.conj()], p)[0].resolve_conj(), want)      # in place, both conjugate
    n = z.conj().imag.reshape(2, 1)[:, 0:1]
    assert n.is_neg()
    with pytest.raises(ValueError):
        rt.beam_reorder([n[:1]], p[:, :1], out=[torch.empty((1, 1), device="cuda")])


def test_lazily_negated_numbers(rt):
    """One number a row, so that the view's strides do not ask for a copy."""
    z = torch.complex(torch.zeros((1, 1), device="cuda"), torch.tensor([[3.0]], device="cuda"))
    x = z.conj().imag
    assert x.is_neg() and float(x) == -3.0
    r = rt.Readout4.quantize(torch.full((1, 1, 1, 40), 7.0, device="cuda"))
    assert torch.all(r.matvec(x) == -21.0)
    logits, scores = torch.zeros((1, 1, 4), device="cuda"), x
    got = rt.beam_select(logits, scores, 1)[0]
    assert torch.allclose(got, torch.full_like(got, -3.0 - 1.3862944), rtol=1e-6, atol=0)
    w = rt.Readout4.quantize(z.conj().imag.view(1, 1, 1, 1) * 1)
    assert torch.all(w.matvec(torch.ones((1, 1), device="cuda")) < 0)
    one = rt.Readout4.quantize(torch.ones((1, 1, 1, 1), device="cuda"))
    with pytest.raises(ValueError, match="out must be"):
        one.matvec(torch.ones((1, 1), device="cuda"), out=z.conj().imag.view(1, 1, 1))
