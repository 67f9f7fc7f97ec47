"""GPU: token sampling against its definition in 64 bits.

Tokens are compared exactly: the weights' relative error (below 1e-13) moves a
border between two tokens past a given random number with a probability below
1e-9 a row.  A log probability is off by its fp32 sum: exponentials exact to two
steps (4 of 2^-24), up to 8 + 60 additions in a thread (4 + 20 at the sizes
here), 9 over a block, 5 over a cluster and 2 steps of the logarithm - at most
72 of 2^-24 relative here, the same absolutely after the logarithm - and by half
a step of its own."""
import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def sample_row(x, T, k, p, min_p, u):
    """The definition for one row in 64 bits."""
    x = x.astype(np.float64)
    if not (0 <= T <= float(np.float32(1e30))) or not p >= 0 or not 0 <= min_p <= 1 or not 0 <= u < 1:
        return -1, math.nan, 2
    if np.isnan(x).any() or x.max() == np.inf:
        return -1, math.nan, 1
    top = x.max()
    if top == -np.inf:
        return -1, math.nan, 4
    if T == 0:
        token = int(np.argmax(x))
    else:
        with np.errstate(over='ignore', under='ignore'):
            w = np.exp((x - top) / T)
        order = np.argsort(-x, kind='stable')
        order = order[(w[order] >= min_p) & (x[order] > -np.inf)]
        if 0 < k < len(order):
            order = order[:k]
        if p < 1:
            cum = np.cumsum(w[order])
            order = order[:1 + int(np.searchsorted(cum[:-1], p * cum[-1]))]
        kept = np.sort(order)
        cum = np.cumsum(w[kept])
        token = int(kept[np.searchsorted(cum, u * cum[-1], side='right')])
    with np.errstate(under='ignore'):
        logp = x[token] - top - math.log(np.exp(x - top).sum())
    return token, logp, 0


def run(native, logits, T=None, k=None, p=None, min_p=None, u=None, want_logp=True):
    m = logits.shape[0]
    f = lambda v, dtype: None if v is None else torch.as_tensor(v, dtype=dtype).expand(m).contiguous().to(DEV)  # noqa: E731
    tokens = torch.full((m,), -7, dtype=torch.int32, device=DEV)
    logp = torch.full((m,), 7.0, device=DEV) if want_logp else None
    flags = torch.zeros(1, dtype=torch.int32, device=DEV)
    native.sample_launch(logits, f(T, FP32), f(k, torch.int32), f(p, FP32), f(min_p, FP32),
                         f(0.5 if u is None else u, FP32), tokens, logp, flags)
    return tokens, logp, flags


def check(native, logits, T=None, k=None, p=None, min_p=None, u=None):
    m = logits.shape[0]
    tokens, logp, flags = run(native, logits, T, k, p, min_p, u)
    x = logits.double().cpu().numpy()
    par = [np.broadcast_to(np.asarray(torch.as_tensor(d if v is None else v, dtype=FP32).double()), (m,))
           for v, d in ((T, 1.0), (p, 1.0), (min_p, 0.0), (u, 0.5))]
    ks = np.broadcast_to(np.asarray(0 if k is None else k), (m,))
    tokens, logp, want_flags = tokens.cpu().numpy(), logp.cpu().numpy(), 0
    for r in range(m):
        token, lp, flag = sample_row(x[r], par[0][r], int(ks[r]), par[1][r], par[2][r], par[3][r])
        want_flags |= flag
        assert tokens[r] == token, (r, tokens[r], token)
        if math.isnan(lp):
            assert math.isnan(logp[r])
        else:
            assert abs(logp[r] - lp) <= 72 * 2.0 ** -24 + 2.0 ** -24 * abs(lp), (r, logp[r], lp)
    assert int(flags) == want_flags


def logits_of(m, vocab, dtype, seed, spread=2.0, head=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((m, vocab), generator=gen) * spread
    if head:
        at = torch.randint(0, vocab, (m, head), generator=gen)
        x.scatter_(1, at, 16.0 - 2.0 * torch.arange(1, head + 1).float().log().expand(m, head))
    return x.to(dtype).to(DEV)


def uniform(m, seed):
    return torch.rand(m, generator=torch.Generator().manual_seed(seed))


SETTINGS = [dict(), dict(T=0.7), dict(k=5), dict(k=300), dict(p=0.9), dict(p=0.2), dict(min_p=0.1), dict(T=0.0),
            dict(T=1.5, k=50, p=0.8), dict(T=0.6, k=1000, p=0.95, min_p=0.01), dict(T=30.0, p=0.5),
            dict(T=30.0, k=777), dict(T=0.01, p=0.9), dict(k=1), dict(p=0.0), dict(min_p=1.0), dict(p=0.99999)]


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('vocab', [1, 2, 7, 33, 1003, 4099])
def test_small_vocabularies(native, vocab, dtype):
    for i, s in enumerate(SETTINGS):
        check(native, logits_of(9, vocab, dtype, i), u=uniform(9, 100 + i), **s)


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('head', [0, 100])
def test_settings(native, dtype, head):
    for i, s in enumerate(SETTINGS):
        check(native, logits_of(3, 50257, dtype, i, head=head), u=uniform(3, i), **s)


@pytest.mark.parametrize('m,vocab,dtype', [(1, 248320, BF16), (2, 248320, FP32), (20, 248320, BF16),
                                           (1, 524288, FP32), (2, 524287, FP16), (1, 500000, FP32),
                                           (70, 65536, FP32), (500, 256, BF16), (160, 40000, FP32), (300, 30000, BF16)])
def test_sizes(native, m, vocab, dtype):
    """One to sixteen CTAs a row, with rows enough to fill the GPU and without."""
    x = logits_of(m, vocab, dtype, 3, head=64)
    for i, s in enumerate((dict(), dict(T=0.8, k=40, p=0.95), dict(T=2.0, p=0.9), dict(T=1.2, k=20000, min_p=1e-6))):
        check(native, x, u=uniform(m, i), **s)


def test_lists_of_every_length(native):
    """Kept sets around the sizes where one CTA ranks them (a few, half a list, a whole one) and beyond."""
    for dtype in (BF16, FP16, FP32):
        x = logits_of(2, 100003, dtype, 21, spread=1.0)
        for i, k in enumerate((2, 100, 255, 256, 257, 700, 1023, 1024, 1025, 3000)):
            check(native, x, k=k, u=uniform(2, i))
            check(native, x, T=1.7, k=k, p=0.9, u=uniform(2, 50 + i))
        peaked = logits_of(2, 100003, dtype, 22, head=1500)
        for i, p in enumerate((0.3, 0.6, 0.8, 0.9, 0.95, 0.99, 0.999)):
            check(native, peaked, T=1.0, p=p, u=uniform(2, i))


def test_estimates_that_fail(native):
    """Nucleus borders where a bin's middle says little of its mass: few heavy tokens at a bin's edge."""
    for dtype in (FP16, FP32):
        x = torch.full((4, 30000), -3.0)
        x[0, 17::1000] = 16.01                         # thirty equal tokens at the bottom of a wide bin
        x[1, 5], x[1, 6:300] = 63.99, 63.6             # one at the top of a bin, others below
        x[2, :20000] = 8.0 + torch.arange(20000) / 1e5  # one bin holds nearly everything
        x[3, ::2] = 1.0
        x = x.to(dtype).to(DEV)
        for i, p in enumerate((0.1, 0.5, 0.75, 0.9, 0.97)):
            for T in (0.3, 1.0, 2.5):
                check(native, x, T=T, p=p, u=uniform(4, i))


@pytest.mark.parametrize('vocab', [261113, 261114])
def test_largest_shares_of_equal_logits(native, vocab):
    """One CTA takes as many bf16 logits as its four counts of 16 bits hold, and one more takes two CTAs."""
    x = torch.full((150, vocab), 1.5, dtype=BF16, device=DEV)
    x[1::4, ::2] = -2.0
    x[2::4, 65280:] = -float('inf')
    x[3::4, :-5] = -float('inf')
    for i, s in enumerate((dict(), dict(p=0.9), dict(k=200000), dict(T=2.0, p=0.3))):
        check(native, x, u=uniform(150, i), **s)


@pytest.mark.parametrize('dtype', [FP16, FP32])
def test_large_nuclei_of_large_batches(native, dtype):
    """Nuclei whose border lies among a few thousand tokens of a CTA that are kept apart, among more than it keeps,
    among equal logits, and below a cut by number."""
    m, vocab = 150, 40009
    x = logits_of(m, vocab, FP32, 51)
    x[1::5] = (x[1::5] * 4).round() / 4            # many equal
    x[2::5] = 2.0 + x[2::5] / 1000                 # all in one or two bins
    x[3::5, ::2] = -float('inf')
    x[4::5] = (x[4::5] > 1.0).float()              # two values
    x = x.to(dtype)
    for i, s in enumerate((dict(p=0.9), dict(p=0.5, T=1.7), dict(p=0.99), dict(k=20000, p=0.8), dict(k=9000, p=0.95, T=3.0),
                           dict(p=0.7, min_p=0.01))):
        check(native, x, u=uniform(m, 60 + i), **s)
        check(native, x[:, 1:], u=0.0, **s)


def test_rows_further_apart_than_32_bits(native):
    vocab, stride = 70001, 2 ** 31 + 17
    for dtype in (BF16, FP16):
        x = torch.empty(2 * stride + vocab, dtype=dtype, device=DEV).as_strided((3, vocab), (stride, 1))
        x.copy_(logits_of(3, vocab, dtype, 41, head=64))
        for i, s in enumerate((dict(), dict(k=30, p=0.9), dict(p=0.99), dict(T=0.0))):
            check(native, x, u=uniform(3, i), **s)


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
def test_values_outside_the_counted_range(native, dtype):
    """Logits of 128 and more, of -128 and less that still have a weight, and near zero, also on a border."""
    base = logits_of(6, 9001, dtype, 31, spread=1.0)
    x = base.clone()
    x[0] += 200.0
    x[1, ::3] = -300.0
    x[2, 4000] = 127.5
    x[3] = (base[3].float() * 2.0 ** -11).to(dtype)            # all below 2^-10 but a few
    x[4, 100:130] = torch.linspace(-9e-4, 9e-4, 30, device=DEV).to(dtype)
    x[5] = torch.where(base[5] > 0.5, base[5], 0.0 * base[5])  # half of the row is 0 or -0
    for i, s in enumerate((dict(), dict(T=100.0), dict(T=100.0, k=3500), dict(T=50.0, p=0.6), dict(k=4400), dict(k=4510),
                           dict(p=0.4), dict(p=0.75), dict(T=0.0), dict(T=20.0, min_p=0.9), dict(min_p=0.999))):
        check(native, x, u=uniform(6, i), **s)


def test_row_parameters(native):
    m = 48
    gen = torch.Generator().manual_seed(5)
    r = lambda: torch.rand(m, generator=gen)  # noqa: E731
    T = torch.where(r() < 0.2, 0.0, 2 * r())
    k = torch.where(r() < 0.3, 0.0, torch.exp(r() * 8)).int()
    k[0], k[1] = -5, 2 ** 31 - 1
    p = torch.where(r() < 0.3, 1.5, r())
    min_p = torch.where(r() < 0.5, 0.0, 0.5 * r())
    check(native, logits_of(m, 32003, BF16, 1, head=30), T, k, p, min_p, r())


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
def test_ties(native, dtype):
    """Rows of few distinct logits: a border inside thousands of equal values goes by index."""
    x = logits_of(6, 70001, FP32, 8).round().to(dtype)
    x[1] = 0.25                                                     # one value
    x[2] = torch.where(x[2] > 3, 1.0, 0.0).to(dtype)                # two
    for i, s in enumerate((dict(k=1), dict(k=35000), dict(k=70000), dict(p=0.5), dict(p=0.25, k=60001),
                           dict(T=0.5, p=0.9), dict(min_p=0.3, p=0.7), dict(T=3.0, k=2000, p=0.5), dict())):
        check(native, x, u=uniform(6, i), **s)
    # an even row cut in half: the border falls exactly between two tokens
    even = torch.zeros((1, 1000), dtype=dtype, device=DEV)
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        assert int(run(native, even, p=0.5, u=u)[0]) == int(500 * u)


def test_random_numbers_at_the_ends(native):
    last = 1 - 2.0 ** -24
    for dtype in (BF16, FP32):
        x = logits_of(4, 9973, dtype, 2, spread=20.0)
        for u in (0.0, 2.0 ** -30, last):
            for s in (dict(), dict(p=0.9), dict(k=3), dict(T=5.0, p=0.999)):
                check(native, x, u=u, **s)


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
def test_masks(native, dtype):
    lowest = torch.finfo(dtype).min
    base = logits_of(8, 20011, dtype, 4)
    gone = torch.rand(base.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    for mask in (-math.inf, lowest):
        x = base.clone()
        for r, share in enumerate((0.0, 0.5, 0.99, 0.9999)):
            x[r] = torch.where(gone[r] < share, mask, x[r].float()).to(dtype)
        x[4, 1:] = mask                       # the first token alone
        x[5, :-1] = mask                      # the last
        x[6] = mask                           # nothing left, or all alike
        x[7, 100:] = -math.inf
        x[7, :50] = lowest                    # both masks
        for i, s in enumerate((dict(), dict(k=50), dict(p=0.9), dict(T=0.0), dict(min_p=0.2), dict(T=1e5, k=10),
                               dict(T=1e5, p=0.5), dict(T=1e30), dict(T=1e-30, p=0.5), dict(T=1e30, k=15000, p=0.3))):
            check(native, x, u=uniform(8, i), **s)


def test_bad_rows_are_refused_alone(native):
    x = logits_of(12, 5000, FP32, 6)
    x[1, 4999], x[3, 0], x[5] = math.nan, math.inf, -math.inf
    T, p, min_p, u = torch.ones(12), torch.full((12,), 0.9), torch.zeros(12), uniform(12, 3)
    check(native, x[[0, 1]], T[:2], p=p[:2], u=u[:2])
    check(native, x[[0, 3]], T[:2], p=p[:2], u=u[:2])
    check(native, x[[0, 5]], T[:2], p=p[:2], u=u[:2])
    for name, value in (('T', -1.0), ('T', math.nan), ('T', math.inf), ('p', -0.1), ('p', math.nan),
                        ('min_p', 1.5), ('min_p', math.nan), ('min_p', -0.1), ('u', 1.0), ('u', -0.5),
                        ('u', math.nan)):
        par = dict(T=T.clone(), p=p.clone(), min_p=min_p.clone(), u=u.clone())
        par[name][7] = value
        check(native, x, **par)


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
def test_strides_and_alignment(native, dtype):
    """Rows that start anywhere inside a 16-byte vector, out of a wider tensor whose other values are NaN."""
    wide = torch.full((5, 3050), math.nan, dtype=dtype, device=DEV)
    values = logits_of(5, 3001, dtype, 9)
    for offset in range(0, 9):
        wide.fill_(math.nan)
        view = wide[:, offset:offset + 3001]
        view.copy_(values)
        for s in (dict(), dict(k=20, p=0.9), dict(T=0.0)):
            check(native, view, u=uniform(5, offset), **s)
    check(native, wide[2:3, 8:3009], u=[0.3])


def test_same_token_whatever_the_launch_shape(native):
    """A row alone (many CTAs) and among many (few CTAs)."""
    row = logits_of(1, 131072, FP32, 11)
    many = row.expand(200, -1).contiguous()
    for i, s in enumerate((dict(), dict(T=1.3, p=0.93), dict(T=2.0, k=9000, p=0.8))):
        u = float(uniform(1, 20 + i))
        one, logp, _ = run(native, row, u=u, **s)
        tokens, _, _ = run(native, many, u=u, **s)
        assert bool((tokens == one).all())


def test_frequencies(native):
    """Tokens come with their probabilities: a stratified set of random numbers hits each token's share exactly."""
    x = logits_of(1, 50, FP32, 12, spread=1.0)
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    tokens, _, _ = run(native, x.expand(n, -1).contiguous(), p=0.8, u=u)
    w = torch.softmax(x.double(), 1)[0].cpu()
    order = w.argsort(descending=True)
    kept = order[:1 + int((w[order].cumsum(0)[:-1] < 0.8).sum())]
    share = torch.zeros(50, dtype=torch.float64)
    share[kept] = w[kept] / w[kept].sum()
    count = torch.bincount(tokens.cpu().long(), minlength=50)
    assert bool(((count - n * share).abs() <= 1).all())   # an interval holds its length in grid points, give or take one


def test_without_logprobs_on_a_stream_and_captured(native):
    x = logits_of(4, 30000, BF16, 13)
    u = uniform(4, 1).to(DEV)
    tokens = torch.zeros(4, dtype=torch.int32, device=DEV)
    logp = torch.zeros(4, device=DEV)
    flags = torch.zeros(1, dtype=torch.int32, device=DEV)
    p = torch.full((4,), 0.9, device=DEV)
    want, want_logp, _ = run(native, x, p=p, u=u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        native.sample_launch(x, None, None, p, None, u, tokens, None, flags)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(tokens, want)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph in graphs:                                    # two graphs over the same buffers
        with torch.cuda.graph(graph):
            native.sample_out(x, None, None, p, None, u, tokens, logp, flags)
    x.copy_(logits_of(4, 30000, BF16, 14))
    want, want_logp, _ = run(native, x, p=p, u=u)
    for graph in graphs:
        tokens.zero_()
        graph.replay()
        assert torch.equal(tokens, want) and torch.equal(logp, want_logp)


def test_no_rows_and_refusals(native):
    x = logits_of(3, 100, FP32, 1)
    u = uniform(3, 1).to(DEV)
    tokens = torch.zeros(3, dtype=torch.int32, device=DEV)
    logp = torch.zeros(3, device=DEV)
    flags = torch.zeros(1, dtype=torch.int32, device=DEV)
    native.sample_launch(x[:0], None, None, None, None, u[:0], tokens[:0], logp[:0], flags)
    good = dict(logits=x, temperature=u, top_k=tokens.clone(), top_p=u, min_p=u, uniform=u, tokens=tokens,
                logprobs=logp, flags=flags)
    native.sample_launch(**good)
    bad = [dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.t()), dict(logits=x[:1].expand(3, 100)),
           dict(logits=x.cpu()), dict(logits=x[:, :0]), dict(logits=torch.zeros((3, (1 << 19) + 1), device=DEV)),
           dict(temperature=u.double()), dict(top_k=tokens.long()), dict(top_p=u[:2]), dict(min_p=u.cpu()),
           dict(uniform=None), dict(uniform=u[:, None]), dict(tokens=tokens.long()), dict(tokens=None),
           dict(logprobs=logp.double()), dict(flags=flags.long()),
           dict(tokens=torch.zeros(6, dtype=torch.int32, device=DEV)[::2])]
    for change in bad:
        with pytest.raises(ValueError):
            native.sample_launch(**{**good, **change})
    with pytest.raises(RuntimeError):
        native.sample_launch(**{**good, 'logprobs': u})     # written over an input


def test_hidden_states_to_tokens(native):
    """The end of a decode step as a server runs it: a 4-bit head in its layer method, then the sampler."""
    method = importlib.import_module('ornith_b200.method')
    runtime = importlib.import_module('ornith_b200.runtime')
    n, k, m = 32000, 2048, 20
    gen = torch.Generator(device=DEV).manual_seed(2)
    codes = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), dtype=torch.int32, device=DEV, generator=gen)
    scales = (0.01 * torch.rand((n, k // 128), device=DEV, generator=gen)).to(BF16)
    layer = torch.nn.Module()
    head = method.W4LinearMethod('head', group=128, logits_fp32=True)
    head.create_weights(layer, k, [n], k, n, BF16, device=DEV)
    layer.w4_codes.weight_loader(layer.w4_codes, codes.view(torch.uint32))
    layer.w4_scales.weight_loader(layer.w4_scales, scales)
    head.process_weights_after_loading(layer)
    rt = runtime.Runtime(['head', 'sampler'], 32, DEV)
    head.bind(rt, 0)
    x = torch.randn((m, k), device=DEV, generator=gen).to(BF16)
    logits = head.apply(layer, x)
    shift = torch.arange(0, 32, 4, dtype=torch.int32, device=DEV)
    weight = (((codes[:, :, None] >> shift) & 15).view(n, k // 128, 128).double() - 8) * scales.double()[:, :, None]
    want = x.double() @ weight.view(n, k).t()
    assert float((logits.double() - want).norm() / want.norm()) < 1e-6   # 200 steps of 2^-24, as a random walk
    check(native, logits, T=0.8, k=50, p=0.95, u=uniform(m, 7))
    tokens = torch.empty(m, dtype=torch.int32, device=DEV)
    native.sample_out(logits, None, None, None, None, uniform(m, 8).to(DEV), tokens, None, rt.slots[1])
    assert bool(((tokens >= 0) & (tokens < n)).all()) and rt.check_error_flags() == [0, 0]


def check_twice(native, x, u, **s):
    """Against the definition, and the same tokens again."""
    first, _, _ = run(native, x, u=u, **s)
    check(native, x, u=u, **s)
    assert torch.equal(first, run(native, x, u=u, **s)[0])


TIED_K, TIED_P = (2, 50, 257, 1000, 1023, 1024), (0.5, 0.9, 0.99, 0.999)


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('vocab', [1500, 70001])
def test_nucleus_border_among_the_ties_of_a_short_top_k(native, dtype, vocab):
    """The k-th logit has more equals than a list holds, and the nucleus ends among them: by index, in every call."""
    x = torch.empty((5, vocab))
    x[0] = 0.25                                                           # one value
    x[1] = torch.where(torch.arange(vocab) % 7 == 3, 1.0, 0.5)            # two
    x[2] = 0.5
    x[2, vocab // 3::2] = -math.inf
    x[2, vocab // 2:vocab // 2 + 40] = torch.linspace(1.0, 3.0, 40)       # a few larger logits above the equal ones
    x[3] = (torch.randn(vocab, generator=torch.Generator().manual_seed(3)) * 40).round() / 40 / 2   # a few hundred
    x[4] = -0.75
    x[4, ::2] = -1.0
    x = x.to(dtype).to(DEV)
    for i, k in enumerate(TIED_K):
        for j, p in enumerate(TIED_P):
            check_twice(native, x, uniform(5, 10 * i + j), k=k, p=p, T=(1.0, 0.7, 3.0)[(i + j) % 3])


@pytest.mark.parametrize('m', [1, 3, 150])
def test_nucleus_border_among_the_ties_of_real_rows(native, m):
    """Ordinary bf16 rows: flat ones, and ones around 20 whose neighbours lie 1/8 apart."""
    vocab = 248320
    x = logits_of(3, vocab, BF16, 71)
    x[1] = (x[1].float() + 12.0).to(BF16)
    x[2] = (x[2].float() * 0.5 + 20.0).to(BF16)
    x = x[torch.arange(m) % 3].contiguous()
    for i, (k, p) in enumerate(((1000, 0.95), (1000, 0.99), (1024, 0.95), (1024, 0.99), (1023, 0.999), (1024, 0.99999))):
        u = uniform(3, 80 + i)[torch.arange(m) % 3]
        if m <= 3:
            check_twice(native, x, u, k=k, p=p)
        else:                                # every copy of a row as it is alone
            many, logp, flags = run(native, x, k=k, p=p, u=u)
            few, few_logp, _ = run(native, x[:3], k=k, p=p, u=u[:3])
            assert torch.equal(many, few[torch.arange(m) % 3]) and int(flags) == 0


def test_tied_rows_alone_and_among_many(native):
    for value, dtype in ((0.25, BF16), (20.0, BF16), (-3.0, FP16)):
        row = torch.full((1, 5000), value, dtype=dtype, device=DEV)
        many = row.expand(200, -1).contiguous()
        for k, p in ((50, 0.9), (1024, 0.5), (1000, 0.999)):
            u = float(uniform(1, k))
            one, _, _ = run(native, row, k=k, p=p, u=u)
            kept = math.ceil(float(np.float32(p)) * k)
            assert int(one) == int(kept * u)                     # equal weights: indices 0 .. kept - 1
            assert bool((run(native, many, k=k, p=p, u=u)[0] == one).all())


def test_logits_a_step_of_the_smallest_number_apart(native):
    """Thousands of different logits inside a range that has no reciprocal in fp32: each round of the search has to
    leave a share of them, not all but one."""
    def steps(vocab, seed):
        order = torch.randperm(vocab, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        return order.view(FP32).to(DEV)[None]                    # 0, 1, 2 ... times 2^-149

    x = torch.cat([steps(20011, 1), -steps(20011, 2), steps(20011, 3)])
    x[2, ::3] *= -1
    for i, s in enumerate((dict(k=9000), dict(p=0.5), dict(k=15000, p=0.3), dict(T=2.0 ** -137, p=0.7), dict(T=2.0 ** -137, k=5000))):
        check(native, x, u=uniform(3, 90 + i), **s)
    large, u = steps(1 << 19, 4), 0.625
    run(native, x, k=9000)                                       # the kernel is loaded
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    token, _, _ = run(native, large, k=1 << 18, u=u)
    end.record()
    end.synchronize()
    kept = torch.arange(1 << 19, device=DEV)[large[0].view(torch.int32) >= 1 << 18]
    assert int(token) == int(kept[int(u * (1 << 18))])           # equal weights, in order of the indices
    assert begin.elapsed_time(end) < 100                         # some 0.2 ms; one value a round would take seconds


@pytest.mark.parametrize('vocab', [300, 1003, 9001, 50257])
def test_log_probability_beside_many_tiny_logits(native, vocab):
    """bf16 logits below 2^-10 share a count, but not an exponential: their sum is the model's all the same."""
    gen = torch.Generator().manual_seed(vocab)
    x = torch.full((6, vocab), -9.0)
    few = min(250, vocab - 20)
    x[:, :few] = 9.6e-4                                            # all on one side of zero
    x[1, :few] = -9.6e-4
    x[2, :few] = (torch.rand(few, generator=gen) * 2 - 1) * 9.7e-4
    x[3, :few // 2] = 0.0
    x[4:, :few] = torch.rand((2, few), generator=gen) * 9.7e-4
    x[:, few + 3] = torch.tensor([0.01, 0.01, 0.002, 1.0, 3.0, 0.5])
    x = x[:, torch.randperm(vocab, generator=gen)].to(BF16).to(DEV)
    for i, s in enumerate((dict(), dict(T=0.7), dict(k=20), dict(p=0.9), dict(k=700, p=0.99), dict(T=0.0), dict(min_p=0.99))):
        check(native, x, u=uniform(6, 110 + i), **s)


def check_logprob(native, x, u, **s):
    """A log probability is computed in 64 bits and rounded once: half a step of its own, 2^-24 relative.  Beside that
    (a) exponentials from a table and the logarithm are off by 1e-12; (b) the sum of an uncut fp16 or fp32 row at T = 1 is that
    of weights in units of 2^-s, each off by half of one; (c) other fp16 and fp32 rows take the logits of more than 2
    below their CTA's largest through fp32: off by 2^-24 for each unit of the difference, 4 times that for the
    exponential and 7 for a vector's sum, each of the logit's own share."""
    tokens, logp, _ = run(native, x, u=u, **s)
    x64 = x.double().cpu()
    vocab = x.shape[1]
    diff = x64 - x64.max(1, keepdim=True).values
    e = diff.exp()
    at = tokens.long().cpu()[:, None]
    assert bool((at >= 0).all())
    others = torch.where(torch.arange(vocab)[None] == at, 0.0, (x64 - x64.gather(1, at)).exp()).sum(1)
    want = -torch.log1p(others)
    slack = torch.full_like(want, 1e-12)
    if x.dtype != BF16:
        slack += vocab * 2.0 ** -(min(51, 62 - (vocab - 1).bit_length()) + 1)
        if s:
            slack += (torch.where(diff < -2, e * (11 - diff.clamp_min(-100)), 0.0).sum(1) / e.sum(1)) * 2.0 ** -24
    err = (logp.double().cpu() - want).abs()
    tol = 2.0 ** -24 * want.abs() + slack
    assert bool((err <= tol).all()), f'off by {float((err / tol).max()):.3g} of the bound'


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('m,vocab', [(60, 700), (24, 4099), (40, 50257), (8, 248320)])
def test_log_probability_to_half_a_step(native, dtype, m, vocab):
    for i, s in enumerate((dict(), dict(T=0.7), dict(p=0.9), dict(T=1.4, k=50, p=0.95), dict(T=0.0), dict(min_p=0.05),
                           dict(k=3000), dict(T=2.0))):
        x = logits_of(m, vocab, dtype, 120 + i, spread=(2.0, 5.0)[i % 2], head=min(vocab // 4, 64))
        check_logprob(native, x, uniform(m, 130 + i), **s)
    if dtype is BF16:                                        # the way of rows that the counts do not hold
        check_logprob(native, (x.float() + 130.0).to(BF16), uniform(m, 140))


def test_hidden_states_to_tokens_captured(native):
    """The same step as a server captures it: the head's method and the sampler in one graph, replayed on new rows."""
    method = importlib.import_module('ornith_b200.method')
    runtime = importlib.import_module('ornith_b200.runtime')
    n, k, m = 32000, 2048, 20
    gen = torch.Generator(device=DEV).manual_seed(12)
    layer = torch.nn.Module()
    head = method.W4LinearMethod('head', group=64, logits_fp32=True)
    head.create_weights(layer, k, [n], k, n, BF16, device=DEV)
    codes = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), dtype=torch.int32, device=DEV, generator=gen)
    layer.w4_codes.weight_loader(layer.w4_codes, codes.view(torch.uint32))
    layer.w4_scales.weight_loader(layer.w4_scales, (0.01 * torch.rand((n, k // 64), device=DEV, generator=gen)).to(BF16))
    head.process_weights_after_loading(layer)
    rt = runtime.Runtime(['head', 'sampler'], 32, DEV)
    head.bind(rt, 0)
    x = torch.randn((m, k), device=DEV, generator=gen).to(BF16)
    T, p, u = torch.full((m,), 0.8, device=DEV), torch.full((m,), 0.95, device=DEV), uniform(m, 1).to(DEV)
    tokens, logp = torch.empty(m, dtype=torch.int32, device=DEV), torch.empty(m, device=DEV)
    head.apply(layer, x)                                         # loaded before the capture
    native.sample_out(head.apply(layer, x), T, None, p, None, u, tokens, logp, rt.slots[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = head.apply(layer, x)
        native.sample_out(logits, T, None, p, None, u, tokens, logp, rt.slots[1])
    for seed in (2, 3):
        x.copy_(torch.randn((m, k), device=DEV, generator=gen).to(BF16))
        u.copy_(uniform(m, seed))
        tokens.fill_(-7)
        graph.replay()
        eager = head.apply(layer, x)
        assert torch.equal(logits, eager)
        want, want_logp, _ = run(native, eager, T=0.8, p=0.95, u=uniform(m, seed))
        assert torch.equal(tokens, want) and torch.equal(logp, want_logp)
        check(native, eager, T=0.8, p=0.95, u=uniform(m, seed))
    assert rt.check_error_flags() == [0, 0]


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
def test_the_lightest_tokens_of_a_zero_random_number(native, dtype):
    """u = 0 draws the first kept token that has a weight in 64 bits, down to the smallest."""
    x = torch.full((4, 700), -10.0)
    x[:, 500] = 64.0
    x[0, 2], x[0, 5] = -10.5, -10.0
    x[1, 2], x[1, 5] = -10.375, 8.0
    x[2, 2], x[2, 5] = -10.4375, 8.0
    x[3] = -30.0
    x[3, 500] = 64.0
    x = x.to(dtype).to(DEV)
    x[:, :2] = -math.inf
    # 2^-1075 is e^-745.133: at T = 0.1 a difference of 74.51, so -10.5 (74.5) has a weight, and -30 (94) none
    for s in (dict(T=0.1), dict(T=0.1, k=600), dict(T=0.1, p=1.0, min_p=0.0), dict(T=0.1, k=699)):
        check(native, x, u=0.0, **s)
        tokens, _, _ = run(native, x, u=0.0, **s)
        if 'k' not in s:
            assert tokens.tolist() == [2, 2, 2, 500]


def test_two_streams_and_one_flag_word(native):
    """Calls that overlap on two streams share nothing but the flag word they are given."""
    x = [logits_of(6, 50257, dtype, 150 + i, head=40) for i, dtype in enumerate((BF16, FP32))]
    x[1][4, 17] = math.nan
    u = uniform(6, 9).to(DEV)
    p = torch.full((6,), 0.9, device=DEV)
    want = [run(native, v, p=p, u=u) for v in x]
    flags = torch.zeros(1, dtype=torch.int32, device=DEV)
    tokens = [torch.zeros((20, 6), dtype=torch.int32, device=DEV) for _ in x]
    logp = [torch.zeros((20, 6), device=DEV) for _ in x]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(20):
        for v, t, lp, side in zip(x, tokens, logp, sides):
            with torch.cuda.stream(side):
                native.sample_launch(v, None, None, p, None, u, t[i], lp[i], flags)
    torch.cuda.synchronize()
    for (token, lp, _), t, out in zip(want, tokens, logp):
        assert bool((t == token).all())
        assert torch.equal(out.nan_to_num(9.0), lp.nan_to_num(9.0).expand(20, -1))
    assert int(flags) == 1


def test_more_rows_than_places(native):
    """A hundred thousand short rows, each with its own settings."""
    m, vocab = 100_003, 37
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn((m, vocab), generator=gen) * 3).to(BF16)
    k = torch.randint(0, 9, (m,), generator=gen, dtype=torch.int32)
    u = torch.rand(m, generator=gen)
    tokens, logp, flags = run(native, x.to(DEV), T=0.75, k=k, u=u)
    w = ((x.double() - x.double().max(1, keepdim=True).values) / 0.75).exp()
    order = x.double().argsort(dim=1, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(1, order, torch.arange(vocab).expand(m, -1).contiguous())
    w = torch.where((k[:, None] < 1) | (rank < k[:, None]), w, 0.0)
    cum = w.cumsum(1)
    target = u.double()[:, None] * cum[:, -1:]
    want = (cum <= target).sum(1)
    clear = ((cum - target).abs() > 1e-9).all(1)              # no border so near that 64 bits tell it otherwise
    assert int(clear.sum()) > 0.999 * m and int(flags) == 0
    assert torch.equal(tokens.cpu().long()[clear], want[clear])
    lp = torch.log_softmax(x.double(), 1).gather(1, tokens.cpu().long()[:, None])[:, 0]
    assert bool(((logp.double().cpu() - lp).abs() <= 2.0 ** -24 * lp.abs() + 1e-12).all())
