"""Token sampling on the GPU against its definition in 64 bits: every row's token has to be equal."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def oracle(logits, u, temperature, top_k, top_p, min_p):
    """The definition, row by row: sort, filter, walk the running weight."""
    rows, vocab = logits.shape
    x = logits.double().cpu().numpy()
    col = lambda v, t: [t(v)] * rows if not torch.is_tensor(v) else [t(i) for i in v.cpu().tolist()]
    f32 = lambda v: float(np.float32(v))
    temperature, top_p, min_p, top_k = col(temperature, f32), col(top_p, f32), col(min_p, f32), col(top_k, int)
    u = u.cpu().numpy()
    out = []
    for r in range(rows):
        if np.isnan(x[r]).any() or (x[r] == -np.inf).all():
            out.append(-1)
            continue
        order = np.lexsort((np.arange(vocab), -x[r]))
        if not temperature[r] > 0:
            out.append(int(order[0]))
            continue
        xs = x[r][order]
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(xs == xs[0], 1.0, np.exp((xs - xs[0]) / temperature[r]))
        w[np.isneginf(xs) | (np.isposinf(xs[0]) & (xs < xs[0]))] = 0.0  # -inf is never drawn, +inf always wins
        if top_k[r] > 0:
            w = w[:top_k[r]]
        if 0 < top_p[r] < 1:
            ahead = np.concatenate(([0.0], np.cumsum(w)[:-1]))
            w = w[ahead <= top_p[r] * w.sum()]
        if min_p[r] > 0:
            w = w[:max(1, int((w >= min_p[r]).sum()))]
        cum = np.cumsum(w)
        over = np.nonzero(cum > float(u[r]) * cum[-1])[0]
        out.append(int(order[over[0] if len(over) else np.nonzero(w > 0)[0][-1]]))
    return torch.tensor(out)


def check(logits, u, **par):
    from multimodal_amd import ops
    par = {"temperature": 1.0, "top_k": 0, "top_p": 0.0, "min_p": 0.0, **par}
    got = ops.sample_tokens(logits.cuda() if not logits.is_cuda else logits, u.cuda(),
                            **{k: v.cuda() if torch.is_tensor(v) else v for k, v in par.items()}).cpu()
    want = oracle(logits, u, **par)
    bad = (got != want).nonzero().flatten().tolist()
    assert not bad, [(r, int(got[r]), int(want[r]), float(u[r])) for r in bad[:5]]
    return got


def logits_for(rows, vocab, dtype, seed=0, sigma=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * sigma).to(dtype), torch.rand(rows, generator=g)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 511, 512, 513, 1000, 8191, 50277, 50304, 65528, 65529, 70001, 131075])
def test_vocabularies(dtype, vocab):
    x, u = logits_for(9, vocab, dtype, vocab)
    check(x, u)
    check(x, u, temperature=0.0)
    check(x, u, temperature=0.7, top_k=40, top_p=0.9)
    check(x, u, top_p=0.5, min_p=0.05)


PAR = [dict(top_k=1), dict(top_k=3), dict(top_k=10 ** 6), dict(top_p=1e-6), dict(top_p=0.3), dict(top_p=0.999), dict(top_p=1.0),
       dict(min_p=1.0), dict(min_p=1e-4), dict(min_p=0.2), dict(temperature=0.05), dict(temperature=1e-30), dict(temperature=50.0),
       dict(temperature=float("inf")), dict(temperature=1.5, top_k=200, top_p=0.8, min_p=0.01), dict(top_k=64, min_p=0.3),
       dict(temperature=0.0, top_k=5, top_p=0.5)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("par", PAR, ids=[str(p) for p in PAR])
def test_parameters(dtype, par):
    x, u = logits_for(40, 3001, dtype, 5)
    check(x, u, **par)


@pytest.mark.parametrize("big", [False, True])
def test_ties_equal_logits_and_borders(big):
    """All weights are 1: the running weight is a whole number, borders are met exactly and ties go to the lowest index."""
    vocab = 70000 if big else 4096
    x = torch.full((8, vocab), 1.5, dtype=BF16)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.125, 2.0 ** -12, 0.3])
    got = check(x, u)
    assert got[0] == 0 and (big or got.tolist()[:4] == [int(4096 * v) for v in (0.0, 0.25, 0.5, 0.75)])
    check(x, u, top_k=17)
    check(x, u, top_p=0.5)
    check(x, u, temperature=0.0)
    x[:, ::3] = -2.0
    check(x, u, temperature=0.25, top_k=5000)
    x[:, 5::7] = 3.0
    check(x, u)


def test_zeros_of_both_signs_tie():
    x = torch.full((16, 300), -0.0, dtype=F16)
    x[:, 1::2] = 0.0
    u = torch.arange(16) / 16.0
    got = check(x, u)
    assert int(got[0]) == 0
    check(x, u, temperature=0.0)
    x[:, 100:] = -1.0
    check(x, u, top_k=120)


def test_infinities_and_nan():
    inf = float("inf")
    x, u = logits_for(12, 700, BF16, 3)
    x[0, :] = -inf                      # nothing to draw
    x[1, 50] = float("nan")
    x[2, 50] = -float("nan")
    x[3, [9, 20, 300]] = inf            # share everything
    x[4, :] = -inf
    x[4, 33] = -4.0                     # one token left
    x[5, 100:] = -inf                   # banned tokens
    x[6, :] = torch.finfo(BF16).min     # the type's lowest value is a value
    x[7, 1:] = torch.finfo(BF16).min
    x[8, :] = torch.finfo(BF16).max
    x[9, :] = -inf
    x[9, [3, 600]] = inf
    for par in (dict(), dict(temperature=0.0), dict(top_k=5, top_p=0.9, min_p=0.01), dict(temperature=float("inf")), dict(temperature=1e-38)):
        got = check(x, u, **par)
        assert got[0] == -1 and got[1] == -1 and got[2] == -1 and got[4] == 33 and got[5] < 100


def test_random_numbers_at_and_beyond_the_ends():
    x, _ = logits_for(6, 900, BF16, 8)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan")])
    from multimodal_amd import ops
    got = ops.sample_tokens(x.cuda(), u.cuda(), top_k=4).cpu()
    order = torch.sort(x.double(), dim=1, descending=True, stable=True)[1]
    assert got[0] == order[0, 0] and got[1] == order[1, 3] and got[2] == order[2, 3] and got[3] == order[3, 3]
    assert got[4] == order[4, 0] and got[5] == order[5, 3]


def test_parameters_per_row_and_strided_rows():
    g = torch.Generator().manual_seed(4)
    rows, vocab = 64, 50277
    wide = (torch.randn(rows, 50304, generator=g) * 2.5).to(BF16)
    wide[:, vocab:] = 100.0             # the padding would win
    u = torch.rand(rows, generator=g)
    par = dict(temperature=torch.rand(rows, generator=g) * 2 * (torch.arange(rows) % 7 != 0),
               top_k=torch.randint(-2, 90, (rows,), generator=g, dtype=torch.int32),
               top_p=torch.rand(rows, generator=g) * 1.2 - 0.1, min_p=torch.rand(rows, generator=g) * 0.1 - 0.02)
    got = check(wide.cuda()[:, :vocab], u, **par)
    assert int(got.max()) < vocab
    # any alignment of the rows' starts
    flat = torch.zeros(20 * 1003 + 8, dtype=F16)
    flat[:] = torch.randn(flat.shape, generator=g).to(F16) * 2
    for shift in range(8):
        x = flat.cuda()[shift:shift + 20 * 1003].view(20, 1003)[:, :1001]
        check(x, torch.rand(20, generator=g), top_p=0.9)


def test_distribution():
    """Frequencies of many draws against softmax, with stratified random numbers."""
    from multimodal_amd import ops
    x, _ = logits_for(1, 61, BF16, 2, sigma=1.0)
    n = 1 << 14
    u = ((torch.arange(n) + 0.5) / n).float()
    tok = ops.sample_tokens(x.cuda().expand(n, 61), u.cuda(), temperature=0.9).cpu()
    p = torch.softmax(x[0].double() / 0.9, 0)
    f = torch.bincount(tok, minlength=61).double()
    assert ((f - n * p).abs() <= 1.0 + 1e-3).all()  # stratified: each interval of length n p holds n p points to within one


def test_replayed_graph_and_other_stream():
    from multimodal_amd import ops
    x, u = logits_for(8, 50304, BF16, 11)
    x, u = x.cuda(), u.cuda()
    out = torch.empty(8, dtype=torch.int64, device="cuda")
    ops.sample_tokens(x, u, top_p=0.9, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.sample_tokens(x, u, top_p=0.9, out=out)
    for rep in range(4):
        x.copy_(logits_for(8, 50304, BF16, 20 + rep)[0])
        u.copy_(torch.rand(8, generator=torch.Generator().manual_seed(rep)))
        want = ops.sample_tokens(x, u, top_p=0.9)
        out.fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.sample_tokens(x, u, top_p=0.9)
    torch.cuda.synchronize()
    assert torch.equal(other, want)


def odd_rows(rows, vocab, dtype, seed, sigma=2.5):
    """Rows that start at any alignment, with values behind them that must not count."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.full((rows * (vocab + 3) + 16,), 60.0, dtype=dtype)
    x = flat[5:5 + rows * (vocab + 3)].view(rows, vocab + 3)[:, :vocab]
    x.copy_((torch.randn(rows, vocab, generator=g) * sigma).to(dtype))
    return flat.cuda()[5:5 + rows * (vocab + 3)].view(rows, vocab + 3)[:, :vocab], torch.rand(rows, generator=g), g


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,vocab", [(1, 500), (257, 504), (257, 505), (257, 506), (300, 1016), (300, 1017), (300, 1018), (1025, 2040),
                                        (1025, 2041), (1025, 2042), (1030, 3), (1030, 64)])
def test_small_vocabularies(dtype, rows, vocab):
    """Every number of rows, at the borders of the vocabularies that are sorted; every filter, parameters of each row."""
    x, u, g = odd_rows(rows, vocab, dtype, rows + vocab)
    check(x, u)
    check(x, u, top_k=20, top_p=0.9)
    check(x, u, temperature=torch.rand(rows, generator=g) * 2 * (torch.arange(rows) % 5 != 0),
          top_k=torch.randint(-2, vocab + 5, (rows,), generator=g, dtype=torch.int32),
          top_p=torch.rand(rows, generator=g) * 1.2 - 0.1, min_p=torch.rand(rows, generator=g) * 0.2 - 0.05)


@pytest.mark.parametrize("par", PAR, ids=[str(p) for p in PAR])
def test_parameters_of_small_vocabularies(par):
    for vocab, rows in ((500, 40), (1010, 270), (2030, 1030)):
        x, u, _ = odd_rows(rows, vocab, BF16, 7)
        check(x, u, **par)


@pytest.mark.parametrize("rows,vocab", [(6, 400), (260, 1000), (1026, 2000)])
def test_ties_infinities_and_nan_of_small_vocabularies(rows, vocab):
    inf = float("inf")
    x, u, _ = odd_rows(rows, vocab, F16, 9)
    x[0, :] = -inf
    x[1, vocab // 2] = float("nan")
    x[2, 50:] = -inf
    x[3, [9, 20, 300]] = inf
    x[4, :] = 0.0
    x[4, ::2] = -0.0
    x[5, :] = 1.5
    for par in (dict(), dict(temperature=0.0), dict(top_k=5, top_p=0.9, min_p=0.01), dict(temperature=inf), dict(top_p=0.5)):
        got = check(x, u, **par)
        assert got[0] == -1 and got[1] == -1 and 0 <= got[2] < 50 and int(got[3]) in (9, 20, 300)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("vocab", [1, 9, 500, 16384, 16385, 50277, 70001])
def test_greedy_rows(dtype, vocab):
    """Ties to the lowest index, zeros of both signs, infinities, NaN; at any alignment."""
    inf = float("inf")
    x, u, g = odd_rows(12, vocab, dtype, vocab)
    at = torch.randint(0, vocab, (12, 3), generator=g)
    for r, v in ((0, 50.0), (1, 50.0), (2, inf), (3, -inf), (4, float("nan")), (5, -float("nan"))):
        if r == 3:
            x[r, :] = -inf
        else:
            x[r, at[r].cuda()] = v
    x[6, :] = -0.0
    x[6, int(at[6, 0])] = 0.0
    x[7, :] = -inf
    x[7, int(at[7, 0])] = -3.0
    x[8, :] = torch.finfo(dtype).min
    got = check(x, u, temperature=0.0)
    assert got[3] == -1 and got[4] == -1 and got[5] == -1 and got[6] == 0 and got[8] == 0 and got[7] == at[7, 0]
    per_row = torch.zeros(12)  # the same through each row's own temperature
    assert torch.equal(check(x, u, temperature=per_row), got)


def ends(rows):
    """Random numbers of 1 and beyond, and NaN (the last token kept), beside the largest below 1 and 0."""
    v = torch.tensor([1.0, float("nan"), 2.0, float("inf"), 1.0, 1 - 2.0 ** -24, 0.0])
    return v.repeat(-(-rows // 7))[:rows]


# at the last one the weights fall below 2^-72 of the largest, which no sum of 64 bits shows
ENDS = [dict(), dict(top_k=3), dict(top_k=5), dict(top_k=11), dict(top_k=200), dict(top_k=500), dict(top_k=700), dict(top_p=0.9),
        dict(min_p=0.01), dict(top_k=11, top_p=0.95, min_p=1e-3), dict(top_k=700, top_p=0.95, min_p=1e-3),
        dict(temperature=0.2, top_k=300), dict(temperature=0.2)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,vocab", [(63, 500), (260, 1010), (1030, 2030), (63, 3001), (28, 50277), (28, 65528), (14, 70001)])
def test_the_last_token_kept_is_drawn_at_one_and_beyond(dtype, rows, vocab):
    """In every kernel: sorted rows, a top-k's list, the histogram, the histogram of long rows."""
    x, _, g = odd_rows(rows, vocab, dtype, vocab + 1)
    for par in ENDS:
        check(x, ends(rows), **par)
    check(x, ends(rows), temperature=0.5 + torch.rand(rows, generator=g), top_k=torch.randint(0, 600, (rows,), generator=g, dtype=torch.int32),
          top_p=0.5 + torch.rand(rows, generator=g), min_p=torch.rand(rows, generator=g) * 0.02)


@pytest.mark.parametrize("rows,vocab", [(28, 500), (260, 1010), (1030, 2030), (28, 3001), (14, 50277), (14, 70001)])
def test_the_last_token_kept_is_never_a_banned_one(rows, vocab):
    """Tokens of -inf have no weight: not drawn at 1 either, also where fewer are left than a top-k would keep."""
    inf = float("inf")
    x, _, g = odd_rows(rows, vocab, F16, vocab + 2)
    some = torch.rand(rows, vocab, generator=g) < 0.5
    x[some.cuda()] = -inf
    x[1, 7:] = -inf
    x[2, :] = -inf
    x[2, vocab // 3] = 0.5
    x[3, [2, vocab // 2, vocab - 1]] = inf   # they share everything
    x[4, :] = torch.finfo(F16).min
    x[8, :] = -0.0
    x[8, 1::2] = 0.0
    for par in ENDS:
        check(x, ends(rows), **par)
