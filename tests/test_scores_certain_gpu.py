"""Scores of rows whose likeliest token has all of the probability: a low temperature, a token that a model is certain of, masks of a finite number. Thousands
of maxima, since what a row's sum of e^(z - maximum) is rounded to depends on the maximum, in every shape that the rows are shared out in."""
import pytest

torch = pytest.importorskip("torch")
from test_token_positions_scores_gpu import BF16, F16, F32, check_scores, gen  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from msnhnet_b200 import tokens
    handle = tokens.TokenOps(0)
    yield handle
    handle.close()


def maxima():
    # (bf16 holds numbers from 32 to 64 in steps of 1/4: some rows are alike there)
    steps = torch.arange(6, 64, 0.125)
    some = torch.tensor([10.0, 15.0, 22.0, 28.0, 100.0])
    spread = 1 + 99 * torch.rand(600, generator=torch.Generator().manual_seed(1))
    return torch.cat([steps, some, -steps[::8], spread]).cuda()


# rows of a call and their length: a warp a row (in one chunk a lane, in more), a block a row, clusters of two, four and eight blocks
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,top", [(1121, 100, 1), (1121, 2048, 5), (1121, 8192, 9), (120, 8200, 3), (60, 16384, 1), (30, 33000, 8), (30, 33000, 0)])
def test_scores_of_rows_with_one_likely_token(ops, dtype, rows, cols, top):
    tops = maxima()
    assert len(tops) >= 1121
    for others in (lambda m: m - 60, lambda m: m - 40, lambda m: torch.full_like(m, -1e4)):
        for first in range(0, 1121, rows):
            m = tops[first:first + rows]
            m = torch.cat([m, tops[:rows - len(m)]]).to(dtype)
            z = others(m.float()).to(dtype)[:, None].expand(rows, cols).contiguous()
            at = torch.randint(0, cols, (rows,), generator=gen(first), device="cuda")
            z.scatter_(1, at[:, None], m[:, None])
            ids = torch.where(torch.arange(rows, device="cuda") % 2 == 0, at, (at + 1) % cols)
            got = logprob, entropy, top_logprobs, top_ids = ops.token_scores(z, ids, top=top)
            assert bool(torch.isfinite(logprob).all()) and bool((logprob <= 0).all())
            assert bool(torch.isfinite(entropy).all()) and bool((entropy >= 0).all())
            if top:
                assert torch.equal(top_ids[:, 0], at) and bool((top_logprobs <= 0).all())
            check_scores(got, z, ids, top, lanes=32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scores_at_a_low_temperature(ops, dtype):
    z = torch.randn(700, 5000, generator=gen(2), device="cuda")
    ids = z.argmax(-1)
    for temperature in (0.2, 0.05, 0.01, 0.001):
        cold = (z / temperature).to(dtype)
        got = ops.token_scores(cold, ids, top=4)
        assert bool(torch.isfinite(got[1]).all()) and bool((got[1] >= 0).all()) and bool((got[2] <= 0).all()) and bool((got[3] >= 0).all())
        check_scores(got, cold, ids, 4)
