"""Drawing where top-k leaves few tokens, or few tokens of a row have weight: rows on both sides of the rules by which the kernel takes its shorter ways, and rows on
which such a way has to be given up.  Tokens are exact, log-probabilities within two roundings of a difference of up to 100 and a logarithm of up to 30 (2e-5)."""
import math

import pytest
import torch

from tests.plain import kv4_plain as plain

pytestmark = pytest.mark.gpu


def _compare(z, k, p=None, m=None, t=None, seed=0):
    from cpmcu_b200.ops.ops import Ops
    ops = Ops(torch.bfloat16)
    rows = z.shape[0]
    u = torch.rand(rows, generator=torch.Generator().manual_seed(seed))
    t = torch.full((rows,), 1.0) if t is None else t
    p = torch.ones(rows) if p is None else p
    m = torch.zeros(rows) if m is None else m
    tok, lp = ops.sample_filtered(z.cuda(), u.cuda(), t.cuda(), k.int().cuda(), p.cuda(), m.cuda())
    for i in range(rows):
        want, logp = plain.sampled(z[i], float(u[i]), float(t[i]), int(k[i]), float(p[i]), float(m[i]))
        assert int(tok[i]) == want, (i, int(tok[i]), want, int(k[i]))
        assert float(lp[i]) == logp or abs(float(lp[i]) - logp) < 2e-5, (i, float(lp[i]), logp)


COUNTS = [1, 2, 3, 31, 32, 50, 127, 128, 129, 200, 223, 224, 225, 255, 256, 257, 500, 1024]


@pytest.mark.parametrize("vocab", [40, 300, 1025, 9000, 32000, 73449])
@pytest.mark.parametrize("rows", [1, 20])
def test_small_top_k(vocab, rows):
    """Counts about the borders, in rows of one and of several blocks, with and without the filters behind them."""
    g = torch.Generator().manual_seed(vocab + rows)
    k = torch.tensor(COUNTS * (2 if rows > 1 else 1))
    n = k.numel()
    z = torch.randn(n, vocab, generator=g) * 3
    p = torch.where(torch.rand(n, generator=g) < 0.5, torch.ones(n), torch.rand(n, generator=g))
    m = torch.where(torch.rand(n, generator=g) < 0.5, torch.zeros(n), 0.2 * torch.rand(n, generator=g))
    t = 0.4 + torch.rand(n, generator=g)
    step = 1 if rows == 1 else n
    for i in range(0, n, step):
        _compare(z[i:i + step], k[i:i + step], p[i:i + step], m[i:i + step], t[i:i + step], seed=i)


def _hard_rows(vocab, g):
    z = torch.randn(10, vocab, generator=g)
    z[0] = 0.25                                                   # all equal: the first k by index
    z[1] = -math.inf
    z[1, 5::vocab // 30] = torch.randn(z[1, 5::vocab // 30].numel(), generator=g)      # fewer tokens with weight than k
    z[2, torch.randperm(vocab, generator=g)[: vocab - 20]] = math.nan                  # most are no numbers
    z[3] = torch.randint(0, 2, (vocab,), generator=g).float()     # two levels
    z[4] = 0.0
    for j in range(0, vocab, 2048):                               # all large tokens beside one another at distances that one thread reads
        z[4, j:j + 4] = 4.0 + torch.rand(z[4, j:j + 4].numel(), generator=g)
    z[5] = -200.0                                                 # one token, and others far below 2^-40 of it
    z[5, vocab // 2] = 0.0
    z[6] = torch.finfo(torch.float32).min
    z[6, ::7] = torch.randn(z[6, ::7].numel(), generator=g)
    z[7, 100:] = -math.inf                                        # what top-k leaves lies in the first block
    z[8, 3] = math.inf
    z[9] = torch.arange(vocab).float() * 1e-4                     # the largest all in the last block
    return z


@pytest.mark.parametrize("vocab", [1100, 20000, 73448])
@pytest.mark.parametrize("k", [2, 60, 200, 224])
def test_rows_that_a_small_top_k_is_not_found_in_at_once(vocab, k):
    z = _hard_rows(vocab, torch.Generator().manual_seed(vocab + k))
    _compare(z, torch.full((10,), k))
    _compare(z, torch.full((10,), k), p=torch.full((10,), 0.7), t=torch.full((10,), 0.3))


@pytest.mark.parametrize("vocab", [700, 20000, 73448])
@pytest.mark.parametrize("spread", [0.2, 1.0, 3.0, 8.0])
def test_mass_alone_where_few_or_many_tokens_have_weight(vocab, spread):
    g = torch.Generator().manual_seed(vocab)
    p = torch.tensor([0.001, 0.3, 0.8, 0.95, 0.9999, 1 - 2.0 ** -24])
    z = torch.randn(6, vocab, generator=g) * spread
    _compare(z, torch.zeros(6), p=p, m=torch.tensor([0.0, 0.0, 1e-6, 0.0, 0.0, 1e-3]))
    z[:, : vocab // 2] -= 100 * spread                            # half of the blocks have nothing
    _compare(z, torch.zeros(6), p=p)


@pytest.mark.parametrize("of_light", [0.5, 0.98, 1.0, 1.02, 2.0])
def test_tokens_at_the_border_of_the_light_ones(of_light):
    """All but one token have a weight about (1 - p) / vocab, below which bins know no tokens."""
    vocab = 30000
    p = torch.tensor([0.5, 0.9, 0.99, 0.7])
    z = torch.zeros(4, vocab)
    for i in range(4):
        z[i, 1:] = math.log(of_light * (1 - float(p[i])) / vocab)
    z[:, 1:] += 1e-3 * torch.rand(4, vocab - 1, generator=torch.Generator().manual_seed(1))
    _compare(z, torch.zeros(4), p=p)
