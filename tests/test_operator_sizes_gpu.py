"""Counts that 32 bits do not hold are refused before anything is copied or allocated for them (tensors of stride 0)."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32, 2 ** 32 + 3])
def test_groups(rt, n):
    x, s = torch.zeros((1, 1, 1), device="cuda"), torch.zeros((1, 1), device="cuda")
    live = torch.ones(1, dtype=torch.int32, device="cuda").expand(n)
    used = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for args in (dict(), dict(live=live)):
        with pytest.raises(ValueError, match="groups"):
            rt.beam_select(x.expand(n, 1, 1), s.expand(n, 1), 1, **args)
    p = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="groups"):
        rt.beam_reorder([torch.zeros((1, 1), device="cuda").expand(n, 1)], p.expand(n, 1))
    assert torch.cuda.max_memory_allocated() - used < 1 << 20


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32, 2 ** 32 + 3])
def test_rows(rt, n):
    r = rt.Readout4.quantize(torch.ones((1, 32, 1, 40), device="cuda"))
    bits, x = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros((1, 32), device="cuda")
    used = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for call in (lambda: r.logits(bits.expand(n, 1)), lambda: r.probabilities(bits.expand(n, 1)),
                 lambda: r.matvec(x.expand(n, 32))):
        with pytest.raises(ValueError, match="rows"):
            call()
    assert torch.cuda.max_memory_allocated() - used < 1 << 20


def test_most_groups_of_one_launch_and_one_more(rt):
    n = 2 * (1 << 20) + 1
    x = torch.randn((n, 1, 3), device="cuda")
    got = rt.beam_select(x, torch.zeros((n, 1), device="cuda"), 1)
    assert torch.equal(got[2][:, 0].long(), x[:, 0].argmax(1))
