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


def _one_of_equal_weights(vocab, g):
    """Rows whose largest logit is not the only token of weight 1, and not the first: differences that a temperature or the exponential rounds away."""
    z = torch.randn(8, vocab, generator=g)
    t = torch.tensor([1.0, 3000.0, 1e9, 1.0, 2e4, 1e30, 1.0, math.inf])
    z[0] *= 1e-9
    z[1] *= 1e-4
    z[3] = -1.0
    z[3, vocab // 3:] = -1e-12 * torch.rand(vocab - vocab // 3, generator=g)
    z[4] *= 1e-3
    z[4, ::2] = math.nan
    z[6] = -torch.finfo(torch.float32).tiny * torch.arange(vocab, 0, -1).float()
    return z, t


@pytest.fixture
def weights_of_the_device(monkeypatch):
    """The definition's weights with the device's exponential.  exp(x) lies half a step of fp32 below 1 at x = -2^-25, and between there and -2^-23 an exponential that is
    off by up to a step may or may not give 1: which tokens of a row weigh 1 is then for the function to say, and the host's is another one."""
    exp = torch.exp
    monkeypatch.setattr(torch, "exp", lambda x: exp(x.cuda()).cpu())


@pytest.mark.parametrize("vocab", [1, 2, 40, 1100, 20000, 73448, 250001])
@pytest.mark.parametrize("setting", ["k", "p", "m"])
@pytest.mark.parametrize("counts", [True, False])
def test_one_token_is_the_first_of_those_of_weight_one(vocab, setting, counts, weights_of_the_device):
    """By a top-k of one, by no mass at all, and by a min-p above one; in calls with and without counts; and where the next number's weight is less after all."""
    from cpmcu_b200.ops.ops import Ops
    ops = Ops(torch.bfloat16)
    z, t = _one_of_equal_weights(vocab, torch.Generator().manual_seed(vocab))
    z = torch.cat((z, torch.randn(4, vocab, generator=torch.Generator().manual_seed(1)) * 3))
    t = torch.cat((t, torch.tensor([0.7, 1.0, 2.0, 5.0])))
    rows = z.shape[0]
    u = torch.rand(rows, generator=torch.Generator().manual_seed(2))
    if setting == "k" and not counts:
        pytest.skip("a count")
    k = torch.full((rows,), 1 if setting == "k" else 0)
    p = torch.full((rows,), 0.0 if setting == "p" else 1.0)
    m = torch.full((rows,), 1.5 if setting == "m" else 0.0)
    tok, lp = ops.sample_filtered(z.cuda(), u.cuda(), t.cuda(), k.int().cuda() if counts else None, p.cuda(), m.cuda())
    for i in range(rows):
        want, logp = plain.sampled(z[i], float(u[i]), float(t[i]), int(k[i]), float(p[i]), float(m[i]))
        assert int(tok[i]) == want and (float(lp[i]) == logp or abs(float(lp[i]) - logp) < 2e-5), (i, int(tok[i]), want)


@pytest.mark.parametrize("vocab", [40, 20000])
def test_verification_of_rows_of_one_token(vocab, weights_of_the_device):
    """The same rows as a model's, with drafting probabilities and without: what a row keeps is that token."""
    from cpmcu_b200.ops.ops import Ops
    from tests.test_gpu_drafts import _check_verify, _i32
    ops = Ops(torch.bfloat16)
    g = torch.Generator().manual_seed(vocab)
    z, t = _one_of_equal_weights(vocab, g)
    z, t = z[:7].repeat_interleave(2, 0), t[:7]                   # seven sequences of two tokens
    cu, seq = [2 * i for i in range(8)], [i // 2 for i in range(14)]
    u, accept = torch.rand(14, generator=g), torch.rand(14, generator=g)
    q = torch.softmax(torch.randn(14, vocab, generator=g), 1)
    ids = [0, 0] * 7
    for s in range(7):                                            # what is drafted: the token itself, the largest logit's, or another
        ids[2 * s + 1] = [plain.sampled(z[2 * s], 0.5, float(t[s]), 1, 1.0, 0.0)[0], int(torch.nan_to_num(z[2 * s], -9.0).argmax()), vocab // 2][s % 3]
    settings = (t, torch.ones(7, dtype=torch.int32), torch.ones(7), torch.zeros(7))
    args = dict(logits=z.cuda(), ids=_i32(ids), cu_q=_i32(cu), token_seq=_i32(seq), most=2, uniform=u.cuda(), temperature=t.cuda(), top_k=settings[1].cuda(), top_p=settings[2].cuda(),
                min_p=settings[3].cuda())
    want = dict(z=z, ids=ids, cu=cu, u=u, settings=settings)
    _check_verify(ops.verify_drafts(**args), **want)
    _check_verify(ops.verify_drafts(**args, draft_probs=q.cuda(), accept=accept.cuda()), **want, probs=q, accept=accept)


@pytest.mark.parametrize("vocab", [300, 32000, 73448])
def test_rows_without_a_count_among_others(vocab):
    """Rows of a call that has counts: those whose count is none (0, below, or the vocabulary's size and more) draw what they draw in a call without counts, to the last bit."""
    from cpmcu_b200.ops.ops import Ops
    ops = Ops(torch.bfloat16)
    g = torch.Generator().manual_seed(vocab)
    z, u = (torch.randn(24, vocab, generator=g) * 3).cuda(), torch.rand(24, generator=g).cuda()
    t, p = (0.3 + 1.5 * torch.rand(24, generator=g)).cuda(), torch.where(torch.rand(24, generator=g) < 0.3, torch.ones(24), torch.rand(24, generator=g)).cuda()
    m = torch.where(torch.rand(24, generator=g) < 0.5, torch.zeros(24), 0.1 * torch.rand(24, generator=g)).cuda()
    k = torch.tensor([0, 5, -1, vocab, 60, vocab + 1, 1, 2 ** 31 - 1] * 3).int()
    tokens, logs = ops.sample_filtered(z, u, t, k.cuda(), p, m)
    without, without_logs = ops.sample_filtered(z, u, t, None, p, m)
    none = ((k <= 0) | (k >= vocab)).cuda()
    assert torch.equal(tokens[none], without[none]) and torch.equal(logs[none], without_logs[none])
    for i in range(24):
        want, logp = plain.sampled(z[i].cpu(), float(u[i]), float(t[i]), int(k[i]), float(p[i]), float(m[i]))
        assert int(tokens[i]) == want and abs(float(logs[i]) - logp) < 2e-5
