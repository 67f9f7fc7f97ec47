"""The operators at the end of a decode step, as cases to be timed and compared.

Two operators, each in a plain form (elementary torch operations) and as the calls of `ornith_b200.native`:

  w4       out[m, n] = sum over groups g of s[n, g] * sum over k in g of x[m, k] * (c[n, k] - z[n, g]): matrix-vector
           products of 1 to 16 rows with 4-bit codes c, group scales s and integer zero points z (8 where there are
           none), for dense layers and for the vocabulary head;
  sample   one token for each row of logits: temperature, min-p, top-k and top-p, then the draw by a given random
           number, and the token's log probability under the model.

`own` says which form `run` takes.
"""
import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def _native():
    import importlib
    import __graft_entry__ as graft
    graft.load_package()
    return importlib.import_module('ornith_b200.native')


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _w4(n, k, group, m, dtype='bf16', out=None, zeros=False, strided=False, **named):
    return dict(named, op='w4', n=n, k=k, group=group, m=m, dtype=dtype, out=out or dtype, zeros=zeros,
                strided=strided)


def _sample(m, vocab, dtype, temperature, top_k, top_p, min_p, shape, masked='none', logprobs=True, strided=False,
            **named):
    """temperature, top_k, top_p, min_p: one value for every row, or 'mixed' (each row its own, some rows off).
    shape: 'peaked' (a few hundred likely tokens above the bulk, what a trained model answers with) or 'flat' (no
    head: high entropy).  masked: 'none', 'inf' (a grammar's mask of -inf) or 'lowest' (the type's lowest value)."""
    return dict(named, op='sample', m=m, vocab=vocab, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p,
                min_p=min_p, shape=shape, masked=masked, logprobs=logprobs, strided=strided)


def listed():
    return [
        # the shared expert's down projection for one token: the smallest call, latency alone
        _w4(2048, 512, 128, 1, name='w4_shared_down_m1'),
        # the widest dense projection of a layer for one token, with zero points
        _w4(12288, 2048, 128, 1, zeros=True, name='w4_qkvz_m1'),
        # the same projection for the largest decode batch, fine groups
        _w4(12288, 2048, 32, 16, dtype='fp16', name='w4_qkvz_m16'),
        # the vocabulary head for one token: the largest weight stream, fp32 logits for the sampler
        _w4(248320, 2048, 128, 1, out='fp32', name='w4_head_m1'),
        # the head for a small batch of requests or of draft tokens
        _w4(248320, 2048, 64, 8, zeros=True, name='w4_head_m8'),
        # odd sizes: rows that end inside a tile, a K that is no multiple of 64, rows of a wider tensor
        _w4(5003, 1056, 32, 5, dtype='fp16', zeros=True, strided=True, name='w4_ragged_m5'),
        # one request: latency, the usual truncation
        _sample(1, 248320, 'bf16', 0.7, 20, 0.95, 0.0, 'peaked', name='sample_request_m1'),
        # a few requests that share nucleus sampling on fp32 logits
        _sample(8, 248320, 'fp32', 1.0, 0, 0.9, 0.0, 'peaked', name='sample_nucleus_m8'),
        # a serving batch, every request with its own settings, a grammar's mask, greedy rows among them
        _sample(64, 248320, 'bf16', 'mixed', 'mixed', 'mixed', 'mixed', 'peaked', masked='inf',
                name='sample_mixed_m64'),
        # drawing from the whole distribution (rollouts): no truncation
        _sample(64, 248320, 'fp32', 1.0, 0, 1.0, 0.0, 'peaked', name='sample_whole_m64'),
        # the largest batch at a high temperature on flat rows: nuclei of many thousand tokens
        _sample(256, 248320, 'bf16', 1.2, 0, 0.95, 0.0, 'flat', logprobs=False, name='sample_flat_m256'),
        # a small odd vocabulary out of a padded tensor, banned tokens at the type's lowest value
        _sample(7, 4099, 'fp16', 'mixed', 'mixed', 'mixed', 'mixed', 'flat', masked='lowest', strided=True,
                name='sample_ragged_m7'),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        group = rng.choice([32, 64, 128, 256])
        dtype = rng.choice(['bf16', 'fp16'])
        return _w4(_log_uniform(rng, 16, 65536), group * _log_uniform(rng, 1, 8192 // group), group, rng.randint(1, 16),
                   dtype=dtype, out=rng.choice([dtype, dtype, 'fp32']), zeros=rng.random() < 0.5,
                   strided=rng.random() < 0.3)
    vocab = _log_uniform(rng, 64, 262144)
    m = _log_uniform(rng, 1, min(512, max(1, 60_000_000 // vocab)))
    return _sample(m, vocab, rng.choice(['bf16', 'fp16', 'fp32']), rng.choice(['mixed', 0.6, 1.0, 1.5]),
                   rng.choice(['mixed', 0, _log_uniform(rng, 1, 2000)]), rng.choice(['mixed', 1.0, 0.95, 0.5]),
                   rng.choice(['mixed', 0.0, 0.05]), rng.choice(['peaked', 'flat']),
                   masked=rng.choice(['none', 'inf', 'lowest']), logprobs=rng.random() < 0.6,
                   strided=rng.random() < 0.3)


def work(case):
    if case['op'] == 'w4':
        n, k, m = case['n'], case['k'], case['m']
        groups = n * (k // case['group'])
        return {'bytes': n * k // 2 + groups * (3 if case['zeros'] else 2) + m * k * 2
                + m * n * (4 if case['out'] == 'fp32' else 2), 'flops': 2 * n * k * m}
    m, vocab = case['m'], case['vocab']
    return {'bytes': m * vocab * (4 if case['dtype'] == 'fp32' else 2) + m * (5 * 4 + 4 + 4 * case['logprobs']),
            'flops': 2 * m * vocab}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _rows(m, width, strided):
    """Where row views come from: m rows of `width` values, of a wider tensor where `strided`."""
    return (m, width + 40 if strided else width)


def _w4_inputs(case, seed, dev):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    n, k, group, m = case['n'], case['k'], case['group'], case['m']
    dtype = DTYPES[case['dtype']]
    x = torch.randn(_rows(m, k, case['strided']), device=dev, generator=gen).to(dtype)[:, :k]
    codes = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), dtype=torch.int32, device=dev, generator=gen)
    scales = (0.01 * torch.randn((n, k // group), device=dev, generator=gen).abs()).clamp_min(2 ** -10).to(dtype)
    zeros = None
    if case['zeros']:
        zeros = torch.randint(4, 12, (n, k // group), dtype=torch.uint8, device=dev, generator=gen)
    return x, codes, scales, zeros


def _mixed(value, rows, pick, dev, dtype):
    """A row parameter: `value` for all rows, or what `pick` makes for each."""
    if value == 'mixed':
        return pick.to(dtype)
    return torch.full((rows,), value, dtype=dtype, device=dev)


def _sample_inputs(case, seed, dev):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    m, vocab = case['m'], case['vocab']
    dtype = DTYPES[case['dtype']]

    def rand(*shape):
        return torch.rand(shape, device=dev, generator=gen)

    logits = torch.randn(_rows(m, vocab, case['strided']), device=dev, generator=gen) * 2.0
    if case['shape'] == 'peaked':
        # a head of likely tokens over the bulk: about 1 of 1000 raised, falling like a power of its rank
        head = max(1, vocab // 1000)
        at = torch.randint(0, vocab, (m, head), device=dev, generator=gen)
        rank = torch.arange(1, head + 1, device=dev, dtype=torch.float32)
        raised = 18.0 - 2.0 * rank.log() + 0.7 * torch.randn((m, head), device=dev, generator=gen)
        logits.scatter_reduce_(1, at, raised, 'amax')
    logits = logits.to(dtype)
    if case['masked'] != 'none':
        lowest = -math.inf if case['masked'] == 'inf' else torch.finfo(dtype).min
        share = rand(m, 1)  # some rows lose nearly everything, some hardly anything
        logits.masked_fill_(rand(*logits.shape) < share, lowest)
    logits = logits[:, :vocab]
    t = rand(m)
    temperature = _mixed(case['temperature'], m, torch.where(rand(m) < 0.15, torch.zeros_like(t), 0.2 + 1.4 * t), dev,
                         torch.float32)
    limit = max(2, vocab // 4)
    top_k = _mixed(case['top_k'], m, torch.where(rand(m) < 0.3, torch.zeros_like(t),
                                                 torch.exp(rand(m) * math.log(limit)).floor()), dev, torch.int32)
    top_p = _mixed(case['top_p'], m, torch.where(rand(m) < 0.3, torch.ones_like(t), 0.05 + 0.949 * rand(m)), dev,
                   torch.float32)
    min_p = _mixed(case['min_p'], m, torch.where(rand(m) < 0.5, torch.zeros_like(t), 0.3 * rand(m) ** 2), dev,
                   torch.float32)
    return logits, temperature, top_k, top_p, min_p, rand(m)


def prepare(case, seed):
    dev = torch.device('cuda', torch.cuda.current_device())
    state = dict(case)
    if case['op'] == 'w4':
        x, codes, scales, zeros = _w4_inputs(case, seed, dev)
        state.update(x=x, codes=codes, scales=scales, zero_points=zeros)
        if own:
            # laid out once, when the weights are loaded
            native = _native()
            state.update(native=native, bank=native.w4_pack(codes.view(torch.uint32), scales, zeros),
                         y=torch.empty((case['m'], case['n']), dtype=DTYPES[case['out']], device=dev),
                         flags=torch.zeros(1, dtype=torch.int32, device=dev))
        return state
    state['inputs'] = _sample_inputs(case, seed, dev)
    if own:
        m = case['m']
        state.update(native=_native(), tokens=torch.empty(m, dtype=torch.int32, device=dev),
                     logp=torch.empty(m, dtype=torch.float32, device=dev) if case['logprobs'] else None,
                     flags=torch.zeros(1, dtype=torch.int32, device=dev))
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    if state['op'] == 'w4':
        if own:
            tiles, scales, zeros = state['bank']
            state['native'].w4_launch(state['x'], tiles, scales, zeros, state['y'], state['flags'], state['n'],
                                      state['k'])
            return state['y']
        return _w4_plain(state['x'], state['codes'], state['scales'], state['zero_points'], state['group'],
                         DTYPES[state['out']])
    if own:
        logits, temperature, top_k, top_p, min_p, uniform = state['inputs']
        state['native'].sample_launch(logits, temperature, top_k, top_p, min_p, uniform, state['tokens'],
                                      state['logp'], state['flags'])
        tokens, logp = state['tokens'], state['logp']
    else:
        tokens, logp = _sample_plain(*state['inputs'], state['logprobs'])
    return {'tokens': tokens, 'logprobs': logp} if state['logprobs'] else {'tokens': tokens}


def _w4_plain(x, codes, scales, zeros, group, out_dtype):
    n, words = codes.shape
    shift = torch.arange(0, 32, 4, dtype=torch.int32, device=codes.device)
    weight = ((codes[:, :, None] >> shift) & 15).view(n, words * 8 // group, group).float()
    weight = weight - (8.0 if zeros is None else zeros[:, :, None].float())
    weight = (weight * scales[:, :, None].float()).view(n, words * 8)
    return (x.float() @ weight.t()).to(out_dtype)


def _sample_plain(logits, temperature, top_k, top_p, min_p, uniform, want_logprobs):
    # 64 bits: the draw and the nucleus compare sums of up to 262144 weights with a border between two tokens
    x = logits.double()
    m, vocab = x.shape
    index = torch.arange(vocab, device=x.device)
    top = x.max(dim=1, keepdim=True).values
    usable = (torch.isfinite(top) & ~x.isnan().any(dim=1, keepdim=True))[:, 0]
    shifted = x - torch.where(torch.isfinite(top), top, 0.0)
    warm = torch.where(temperature > 0, temperature, 1.0).double()[:, None]
    weight = torch.exp(shifted / warm)
    weight = torch.where(weight >= min_p.double()[:, None], weight, 0.0)
    by_value, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: lowest index first
    in_order = weight.gather(1, order)
    limit = torch.where(top_k > 0, top_k.long(), vocab)[:, None]
    in_order = torch.where(index[None, :] < limit, in_order, 0.0)
    mass = in_order.cumsum(dim=1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], dim=1)
    p = top_p.double()[:, None]
    keep = (p >= 1) | (before < p * mass[:, -1:]) | (index[None, :] == 0)
    kept = torch.zeros_like(weight).scatter_(1, order, torch.where(keep, in_order, 0.0))
    reached = kept.cumsum(dim=1)
    token = (reached <= uniform.double()[:, None] * reached[:, -1:]).sum(dim=1)
    greedy = torch.where(x == top, index[None, :], vocab).min(dim=1).values
    token = torch.where(temperature > 0, token, greedy)
    token = torch.where(usable, token, -1)
    if not want_logprobs:
        return token.int(), None
    # log p = -log1p(the other weights over the token's): exact to the last bits where p is near 1
    at = token.clamp_min(0)[:, None]
    chosen = shifted.gather(1, at)
    others = torch.where(index[None, :] == at, 0.0, torch.exp(shifted - chosen)).sum(dim=1)
    logp = torch.where(usable, -torch.log1p(others), math.nan)
    return token.int(), logp.float()


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    dev = torch.device('cuda', torch.cuda.current_device())
    if case['op'] == 'w4':
        return _w4_exact(case, *_w4_inputs(case, seed, dev))
    if case['m'] * case['vocab'] > 40_000_000:
        return None  # sorted on the host, one row after the other
    return _sample_exact(case, *(v.double().cpu().numpy() for v in _sample_inputs(case, seed, dev)))


def _w4_exact(case, x, codes, scales, zeros):
    n, k, group, m = case['n'], case['k'], case['group'], case['m']
    y = torch.zeros((m, n), dtype=torch.float64, device=x.device)
    x64 = x.double()
    octets = codes.view(torch.uint8)  # little endian: byte b of a word holds values 2b and 2b + 1
    step = max(1, 2 ** 26 // k)
    for first in range(0, n, step):
        part = octets[first:first + step]
        codes64 = torch.stack([part % 16, part // 16], dim=-1).reshape(part.shape[0], k).double()
        for g in range(k // group):
            of = slice(g * group, (g + 1) * group)
            zero = 8.0 if zeros is None else zeros[first:first + step, g:g + 1].double()
            dot = x64[:, of] @ (codes64[:, of] - zero).t()
            y[:, first:first + step] += dot * scales[first:first + step, g].double()
    return y


def _sample_exact(case, logits, temperature, top_k, top_p, min_p, uniform):
    import numpy as np
    tokens = np.full(case['m'], -1, dtype=np.int32)
    logp = np.full(case['m'], np.nan)
    for r in range(case['m']):
        row = logits[r]
        if np.isnan(row).any() or not np.isfinite(row.max()):
            continue
        best = int(row.argmax())
        if temperature[r] == 0:
            tokens[r] = best
        else:
            live = np.flatnonzero(row > -np.inf)
            with np.errstate(under='ignore'):
                weight = np.exp((row[live] - row[best]) / temperature[r])
            ranked = np.lexsort((live, -row[live]))
            ranked = ranked[weight[ranked] >= min_p[r]]
            if top_k[r] > 0:
                ranked = ranked[:int(top_k[r])]
            if top_p[r] < 1:
                mass = np.cumsum(weight[ranked])
                ranked = ranked[:1 + int(np.searchsorted(mass[:-1], top_p[r] * mass[-1]))]
            chosen = np.sort(ranked)
            mass = np.cumsum(weight[chosen])
            tokens[r] = live[chosen[int(np.searchsorted(mass, uniform[r] * mass[-1], side='right'))]]
        with np.errstate(under='ignore', over='ignore'):
            ratio = np.exp(row - row[tokens[r]])
        ratio[tokens[r]] = 0.0
        logp[r] = -np.log1p(ratio.sum())
    return {'tokens': tokens, 'logprobs': logp} if case['logprobs'] else {'tokens': tokens}
