"""beam_select's scores are float64 up to one rounding: where a score and the logarithm of its beam's sum nearly cancel,
the difference shows how far the sum and the logarithm are off.

Tolerance, u = 2^-53: an exponential is off by 3 u (its argument, at most 1/2 after the first, rounds twice, the
polynomial and its last step once), a sum of up to 32 roundings (a thread's terms, the wave, the waves) by 32 u, the
logarithm of s <= e^12 by 2 ln 2 * 17 u for its own exponential's argument, 2 u beside it and 12 u for its sum, the
differences behind it by 12 u: below 96 u.  Then half a step of the float32 result."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

U = 2.0 ** -53


@pytest.mark.parametrize("win,v", [(1, 100), (8, 480), (4, 1000), (64, 200), (4, 2000), (1, 8192), (9, 1025), (2, 40000)])
@pytest.mark.parametrize("t", [-0.5, -0.49, -0.31, -0.02])
def test_scores_next_to_their_logarithms(rt, win, v, t):
    """One logit of 0 a beam and the others t ln 2 below it, where a short series for 2^t is furthest off."""
    low = np.float32(t * np.log(2.0))
    x = np.full((3, win, v), low, np.float32)
    x[:, :, v // 3] = 0
    n = np.array([v, v, v // 2], np.int32)
    s = 1 + (n - 1).astype(np.longdouble) * np.exp(np.longdouble(low))
    score = np.repeat(np.log(s).astype(np.float32)[:, None], win, 1)
    score[1] += np.float32(1e-5) * np.arange(win, dtype=np.float32)
    got = [a.cpu().numpy() for a in rt.beam_select(torch.from_numpy(x).cuda(), torch.from_numpy(score).cuda(), win,
                                                   live=torch.from_numpy(n).cuda())]
    for g in range(3):
        exact = np.sort((score[g].astype(np.longdouble) - np.log(s[g])))[::-1][:win]
        off = np.abs(got[0][g].astype(np.longdouble) - exact)
        assert np.all(got[2][g] == v // 3)
        assert np.all(off <= 96 * U + np.spacing(np.abs(exact).astype(np.float32)) / 2), float(off.max())
