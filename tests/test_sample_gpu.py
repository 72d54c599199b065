"""EET.sample_rows against a plain restatement in 64 bits."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


def _sample(*args, **kw):
    from eet_b200 import EET
    return EET.sample_rows(*args, **kw)


def kept64(x, temperature, top_k, top_p, min_p):
    """(order of what stays, its weights in 64 bits) of a row, CPU."""
    x = x.double()
    x = torch.where(x.isnan(), -math.inf, x)
    order = torch.sort(x, descending=True, stable=True).indices
    order = order[x[order] > -math.inf]
    if len(order) == 0:
        return order, x[order]
    if not temperature > 0:
        return order[:1], torch.ones(1, dtype=torch.float64)
    top = x[order[0]]
    w = torch.where(x[order] == top, 1.0, torch.exp((x[order] - top) / float(torch.tensor(temperature, dtype=FP32))))
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    n = len(order)
    if top_p < 1:
        front = torch.cat((w.new_zeros(1), w.cumsum(0)[:-1]))
        n = int((front < float(torch.tensor(top_p, dtype=FP32)) * w.sum()).sum())
    if min_p > 0:
        n = min(n, int((w >= min(1.0, float(torch.tensor(min_p, dtype=FP32)))).sum()))
    n = max(n, 1)
    return order[:n], w[:n]


def draw64(x, u, *settings):
    """(token, logprob, how near the draw is to the border of another token, how many weights are not exact) of a row."""
    order, w = kept64(x, *settings)
    if len(order) == 0:
        return -1, -math.inf, 1.0, 0
    index, place = order.sort()
    w = w[place]
    run = w.cumsum(0)
    goal = float(u) * run[-1]
    at = min(int((run <= goal).sum()), len(index) - 1)
    while at > 0 and w[at] == 0:
        at -= 1
    near = float(((run - goal).abs() / run[-1]).min())
    return int(index[at]), float(torch.log(w[at] / run[-1])), near, int((w != 1).sum())


def _check(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens are those of the definition.  Weights are whole multiples of 2^-44 of the largest, so a running sum of n of them that are not equal
    to it is off by up to n 2^-45 of it, which is less than that part of the whole: a draw that lies nearer to a border than 2 n 2^-44 proves
    nothing.  The logarithm is rounded to fp32 once, of a sum that is off by as much."""
    tokens, logprobs = _sample(logits, uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert tokens.dtype == torch.int64 and logprobs.dtype == FP32 and tokens.shape == logprobs.shape == (logits.shape[0],)
    tokens, logprobs = tokens.tolist(), logprobs.double().tolist()
    column = lambda v, r: v[r].item() if torch.is_tensor(v) else v  # noqa: E731
    sure = 0
    for r, x in enumerate(logits.cpu()):
        want, logprob, near, inexact = draw64(x, uniform[r].item(), *(column(v, r) for v in (temperature, top_k, top_p, min_p)))
        if inexact and near <= 2 * inexact * 2.0 ** -44 and uniform[r].item() > 0:
            continue
        sure += 1
        assert tokens[r] == want, (r, tokens[r], want)
        if want >= 0:
            assert abs(logprobs[r] - logprob) <= 2.0 ** -24 * abs(logprob) + x.numel() * 2.0 ** -44 + 1e-12, (r, logprobs[r], logprob)
        else:
            assert logprobs[r] == -math.inf
    assert 10 * sure >= 9 * logits.shape[0]


def _logits(rows, vocab, dtype, seed, spread=2.0, peaks=30):
    gen = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=gen)
    if peaks:
        place = torch.randint(0, vocab, (rows, peaks), generator=gen)
        x.scatter_(1, place, 6 + 3 * torch.rand(rows, peaks, generator=gen))
    return x.to(dtype).cuda(), torch.rand(rows, generator=gen).cuda()


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_k=5000), dict(top_p=0.9), dict(top_p=0.3), dict(min_p=0.05),
            dict(top_k=40, top_p=0.8), dict(top_k=6000, top_p=0.95), dict(temperature=1.7, top_k=100, top_p=0.9, min_p=0.02), dict(temperature=0.0),
            dict(temperature=0.05, top_p=0.99), dict(temperature=30.0, top_p=0.5), dict(top_p=0.0), dict(top_p=1e-9, top_k=3), dict(min_p=1.0)]


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("rows,vocab,dtype", [(1, 32000, FP32), (3, 32001, FP16), (5, 64000, BF16), (160, 1009, FP32), (40, 7, FP16), (2, 1, BF16)])
def test_sample(settings, rows, vocab, dtype):
    _check(*_logits(rows, vocab, dtype, 1), **settings)


@pytest.mark.parametrize("settings", [dict(top_k=5000), dict(top_p=0.9), dict(top_k=20000, top_p=0.6), dict(top_p=0.5, min_p=0.5), dict()])
@pytest.mark.parametrize("kind", ["flat", "equal", "two", "steps", "far"])
@pytest.mark.parametrize("dtype", [FP16, FP32])
def test_sample_where_no_list_holds_the_candidates(settings, kind, dtype):
    """Tens of thousands of values in one bin of the histogram, all of them equal or a few different ones."""
    vocab = 40000
    gen = torch.Generator().manual_seed(4)
    x = {"flat": 1e-4 * torch.randn(2, vocab, generator=gen), "equal": torch.full((2, vocab), 3.25),
         "two": torch.randint(0, 2, (2, vocab), generator=gen).float(), "steps": torch.randint(0, 5, (2, vocab), generator=gen) * 0.001,
         "far": 100.0 - torch.arange(2 * vocab).view(2, vocab) * 0.01}[kind].to(dtype).cuda()
    _check(x, torch.tensor([0.25, 0.8], device="cuda"), **settings)


@pytest.mark.parametrize("settings", [dict(top_k=50, top_p=0.95, temperature=0.3), dict(top_k=20000, temperature=0.05), dict(top_k=1000), dict(top_k=7)])
@pytest.mark.parametrize("spread", [4.0, 60.0, 3000.0])
def test_sample_of_the_most_from_a_row_that_reaches_far_down(settings, spread):
    """Nearly all tokens lie more than 32 factors of e below the largest, some of them masked with the lowest number."""
    logits, uniform = _logits(3, 32000, FP32, 11, spread, peaks=10)
    logits[:, 0] = 10 * spread
    _check(logits, uniform, **settings)
    logits[:, 1000:9000] = torch.finfo(FP32).min
    _check(logits, uniform, **settings)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.4), dict(top_k=2, top_p=0.5)])
def test_sample_among_ties(settings):
    """Equal logits: the lower index stays, also where they lie in different threads and CTAs."""
    x = torch.full((6, 30000), -1.0)
    places = [[0, 29999], [5, 6, 7, 8], [100, 9000, 18000, 27000], [29998, 29999], [0, 1, 2, 15000, 29000], [12345]]
    for row, place in zip(x, places):
        row[place] = 9.0
    x[3, 7] = 9.5
    for u in (0.0, 0.2, 0.499, 0.7, 1 - 2.0 ** -24):
        _check(x.half().cuda(), torch.full((6,), u, device="cuda"), **settings)


def test_sample_of_masked_infinite_and_missing_values():
    lowest = torch.finfo(FP32).min
    x = torch.tensor([[-math.inf] * 4, [math.nan, -math.inf, 2.0, -math.inf], [math.inf, 1.0, math.inf, 5.0], [lowest, lowest, 0.0, lowest],
                      [lowest] * 4, [math.nan] * 4, [-0.0, 0.0, -0.0, 0.0], [1.0, math.nan, math.nan, 1.0]]).cuda()
    for u, settings in itertools.product((0.0, 0.3, 0.6, 0.999), (dict(), dict(top_k=2), dict(top_p=0.4), dict(temperature=0.0), dict(min_p=0.1))):
        _check(x, torch.full((8,), u, device="cuda"), **settings)


def test_sample_of_a_random_number_outside_its_range():
    """The first or the last token that stays, nothing else."""
    x = torch.tensor([[-math.inf, 1.0, 1.0, -math.inf]] * 4).cuda()
    got = _sample(x, torch.tensor([-1.0, math.nan, 1.0, math.inf], device="cuda"))[0]
    assert got.tolist() == [1, 1, 2, 2]


def test_sample_with_settings_of_every_row():
    rows = 33
    logits, uniform = _logits(rows, 5003, BF16, 2)
    gen = torch.Generator().manual_seed(9)
    u = torch.rand(4, rows, generator=gen)
    temperature = torch.where(u[0] < 0.2, torch.zeros(rows), 0.2 + 2 * u[0])
    top_k = torch.where(u[1] < 0.3, torch.zeros(rows), 200 * u[1]).int()
    top_p = torch.where(u[2] < 0.3, torch.ones(rows), u[2])
    min_p = torch.where(u[3] < 0.5, torch.zeros(rows), 0.2 * u[3])
    args = [t.cuda() for t in (temperature, top_k, top_p, min_p)]
    _check(logits, uniform, *args)
    # what is out of range in a tensor leaves all, or the first token
    args = [torch.tensor([v] * rows, device="cuda", dtype=t) for v, t in ((-1.0, FP32), (-5, torch.int32), (7.0, FP32), (-3.0, FP32))]
    assert torch.equal(_sample(logits, uniform, *args)[0], logits.float().argmax(-1))
    args[0].fill_(1.0)
    assert torch.equal(_sample(logits, uniform, *args)[0], _sample(logits, uniform)[0])
    assert torch.equal(_sample(logits, uniform, torch.full_like(uniform, math.nan))[0], logits.float().argmax(-1))


def test_sample_of_strided_and_unaligned_rows():
    base = torch.randn(7, 4001, generator=torch.Generator().manual_seed(5)).half().cuda()
    uniform = torch.rand(7, generator=torch.Generator().manual_seed(6)).cuda()
    for begin, end in ((0, 4001), (1, 4001), (3, 3004), (7, 8), (5, 21)):
        _check(base[:, begin:end], uniform, top_k=30, top_p=0.9)
        _check(base.float()[::2, begin:end], uniform[::2].contiguous(), top_p=0.9)


def test_sample_of_the_largest_vocabulary():
    for dtype, rows in ((FP32, 1), (BF16, 20)):
        logits, uniform = _logits(rows, 1 << 18, dtype, 3)
        _check(logits, uniform, top_p=0.9)
        _check(logits, uniform)


def test_sample_frequencies():
    """Every token comes as often as it should: 4096 numbers spread evenly leave each count within 1 of its probability times 4096 and the
    borders' rounding."""
    x = torch.tensor([[0.3, -1.0, 2.0, 1.1, -math.inf, 0.0, 1.9]]).expand(4096, 7).cuda()
    uniform = ((torch.arange(4096) + 0.5) / 4096).cuda()
    for settings in (dict(), dict(top_k=3), dict(top_p=0.8, temperature=1.3)):
        got = torch.bincount(_sample(x, uniform, **settings)[0].cpu(), minlength=7)
        order, w = kept64(x[0].cpu(), settings.get("temperature", 1.0), settings.get("top_k", 0), settings.get("top_p", 1.0), 0.0)
        want = torch.zeros(7, dtype=torch.float64)
        want[order] = 4096 * w / w.sum()
        assert ((got - want).abs() <= 1).all()


def test_sample_in_a_graph_and_on_another_stream():
    logits, uniform = _logits(4, 32000, FP16, 7)
    top_p = torch.full((4,), 0.9, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = _sample(logits, uniform, top_p=top_p)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            tokens, logprobs = _sample(logits, uniform, top_p=top_p)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(tokens, eager[0]) and torch.equal(logprobs, eager[1])
    uniform.copy_(1 - uniform)
    top_p.fill_(0.5)
    logits.copy_(logits.flip(1))
    graph.replay()
    want = _sample(logits, uniform, top_p=top_p)
    torch.cuda.synchronize()
    assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])


def test_sample_refuses():
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    ones = torch.ones(2, device="cuda")
    for bad in (dict(x=x.double()), dict(x=x.cpu()), dict(x=x[0]), dict(x=x.t()), dict(u=u.double()), dict(u=u[:1]), dict(u=u.cpu()),
                dict(temperature=-0.1), dict(temperature=math.nan), dict(top_k=-1), dict(top_k=1.5), dict(top_p=1.1), dict(top_p=-0.1),
                dict(top_p=math.nan), dict(min_p=1.5), dict(min_p=-1.0), dict(temperature=ones.double()), dict(top_k=ones), dict(top_p=ones[:1]),
                dict(min_p=ones.cpu()), dict(x=torch.zeros(1, (1 << 18) + 1, device="cuda"), u=u[:1]),
                dict(x=torch.zeros(2, 0, device="cuda"))):
        args = dict(x=x, u=u)
        args.update(bad)
        with pytest.raises(RuntimeError, match="sample_rows"):
            _sample(args.pop("x"), args.pop("u"), **args)
    assert _sample(x[:0], u[:0])[0].shape == (0,)
