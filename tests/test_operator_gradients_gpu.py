"""The read-out and beam entry points have no gradient: they refuse what would lose one, and a tensor that they write to
counts as changed for a backward pass that has kept it."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)


def test_scores_that_require_a_gradient(rt):
    x, s = torch.zeros((2, 3, 5), device="cuda"), torch.zeros((2, 3), device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        rt.beam_select(x, s, 2)
    with torch.no_grad():
        rt.beam_select(x, s, 2)
    rt.beam_select(x, s.detach(), 2)


def test_buffers_that_require_a_gradient(rt):
    p = torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device="cuda")
    leaf = torch.arange(4.0, device="cuda").requires_grad_()
    plain = torch.zeros(4, device="cuda")
    inner = (torch.zeros(4, device="cuda").requires_grad_() * 2)
    for args in (([leaf], p), ([plain, leaf], p), ([leaf], p, [plain]), ([plain], p, [inner]), ([inner], p)):
        with pytest.raises(ValueError, match="gradient"):
            rt.beam_reorder(*args)
    assert leaf.tolist() == [0, 1, 2, 3]
    with torch.no_grad():
        rt.beam_reorder([leaf], p)
    assert leaf.tolist() == [1, 0, 3, 3]


def test_written_tensors_count_as_changed(rt):
    p = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    for out in (None, "apart"):
        w = torch.ones(2, device="cuda", requires_grad=True)
        x, y = torch.tensor([1.0, 2.0], device="cuda"), torch.tensor([5.0, 6.0], device="cuda")
        z = (w * x * 1).sum() if out is None else (w * y * 1).sum()
        moved = rt.beam_reorder([x], p, out=None if out is None else [y])
        assert moved[0].tolist() == [2.0, 1.0]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    # what is only read is as it was
    w, x = torch.ones(2, device="cuda", requires_grad=True), torch.tensor([1.0, 2.0], device="cuda")
    z = (w * x).sum()
    rt.beam_reorder([x], p, out=[torch.empty_like(x)])
    z.backward()
    assert w.grad.tolist() == [1.0, 2.0]


def test_out_of_a_read_out(rt):
    r = rt.Readout4.quantize(torch.ones((1, 32, 1, 40), device="cuda"))
    bits, x = torch.full((1, 1), -1, dtype=torch.int32, device="cuda"), torch.ones((1, 32), device="cuda")
    for call in (lambda o: r.logits(bits, out=o), lambda o: r.probabilities(bits, out=o), lambda o: r.matvec(x, out=o)):
        leaf = torch.zeros((1, 1, 40), device="cuda", requires_grad=True)
        with pytest.raises(ValueError, match="gradient"):
            call(leaf)
        assert torch.all(leaf == 0)
        with torch.no_grad():
            call(leaf)
        out, w = torch.zeros((1, 1, 40), device="cuda"), torch.ones(40, device="cuda", requires_grad=True)
        z = (w * out).sum()
        assert call(out) is out
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    with torch.inference_mode():                         # tensors without a version
        out = torch.zeros((1, 1, 40), device="cuda")
        r.matvec(x, out=out)
        rt.beam_reorder([torch.zeros(2, device="cuda")], torch.zeros((1, 2), dtype=torch.int32, device="cuda"))
    r.matvec(x, out=out)
