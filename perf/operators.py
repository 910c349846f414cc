"""Decoding operators of the language core: plain forms, cases and inputs.

Four operators, as a pool of streaming sessions uses them when it decodes with beams:

quantize  values to 8-bit floating point (e4m3) with one fp32 scale for each block of 128
          along k (activations: 1 x 128, weights: 128 x 128)
matmul    the product of two such matrices, y[m][n] = sum_k a[m][k] w[n][k], with a
          projection's bias and memory term as its epilogue
select    beam search's step: the best `beams` of beams x vocabulary, by cumulative log
          probability, from the logits of every beam
reorder   the session states that follow the selected beams, moved in place

Sizes are the projections, states and vocabulary (264) of the language presets (32 columns of
width 768; 64 columns of width 1024), and generic larger ones.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
E4M3_MAX = 448.0
TINY = 2.0 ** -126
BLOCK = 128
PAD = 256   # the byte vocabulary's padding token, which a finished beam repeats
END = 258   # the token that finishes a beam
ADD = 0.25  # the output projection's weight of the region memory


OURS = []   # the framework's modules, imported once as a program does at its start


def package():
    if not OURS:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'neurogen-2.5_b200'))
        from neurogen_b200 import blockscale, decoding
        OURS.extend((blockscale, decoding))
    return OURS


def listed():
    return [
        # One session's hidden state on its way into a projection: latency.
        dict(name='quantize 1 x 768', op='quantize', m=1, k=768, dtype='fp32', rows=1, strided=False),
        # The trace and spike-count features of 2,048 beams, 64 columns.
        dict(name='quantize 2048 x 6400', op='quantize', m=2048, k=6400, dtype='fp32', rows=1, strided=False),
        # A large weight matrix, ragged, quantised once at model load.
        dict(name='quantize weight 8000 x 8100', op='quantize', m=8000, k=8100, dtype='bf16', rows=128, strided=True),
        # Single-token decode: one session's output projection with bias and memory term.
        dict(name='matmul 1 x 768 x 3200', op='matmul', m=1, n=768, k=3200, out='fp32', epilogue=True),
        # 256 sessions' feedback projection of one region.
        dict(name='matmul 256 x 928 x 768', op='matmul', m=256, n=928, k=768, out='fp32', epilogue=False),
        # A ragged batch on sizes that end inside every tile.
        dict(name='matmul 333 x 1001 x 700', op='matmul', m=333, n=1001, k=700, out='bf16', epilogue=True),
        # Generic large product (a long prompt batch): tensor-core bound.
        dict(name='matmul 8192 x 8192 x 4096', op='matmul', m=8192, n=8192, k=4096, out='bf16', epilogue=False),
        # One conversation, four beams: latency.
        dict(name='select 1 x 4 x 264', op='select', groups=1, beams=4, vocab=264, dtype='fp32', masked=False,
             finished=False, strided=False),
        # 256 conversations of 8 beams, some finished, control tokens not allowed.
        dict(name='select 256 x 8 x 264', op='select', groups=256, beams=8, vocab=264, dtype='fp32', masked=True,
             finished=True, strided=False),
        # A word-piece vocabulary, odd, in 16 bits (equal logits are common).
        dict(name='select 16 x 5 x 50001', op='select', groups=16, beams=5, vocab=50001, dtype='bf16', masked=True,
             finished=True, strided=False),
        # One conversation's four states of the tiny preset: latency.
        dict(name='reorder 1 x 4 x 704', op='reorder', groups=1, beams=4, size=704),
        # 256 conversations of 8 beams, 44,032 floats a state.
        dict(name='reorder 256 x 8 x 44032', op='reorder', groups=256, beams=8, size=44032),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['quantize', 'matmul', 'matmul', 'select', 'select', 'reorder'])
    if op == 'quantize':
        m, k = log_int(rng, 1, 8192), log_int(rng, 1, 8192)
        return dict(op=op, m=m, k=k, dtype=rng.choice(list(DTYPES)), rows=rng.choice([1, 1, 128]),
                    strided=rng.random() < 0.5)
    if op == 'matmul':
        m = rng.choice([log_int(rng, 1, 16), log_int(rng, 17, 8192)])
        return dict(op=op, m=m, n=log_int(rng, 16, 8192), k=log_int(rng, 16, 4096), out=rng.choice(list(DTYPES)),
                    epilogue=rng.random() < 0.5)
    if op == 'select':
        beams = rng.randint(1, 32)
        vocab = rng.choice([264, log_int(rng, 260, 200000)])
        groups = log_int(rng, 1, max(1, min(1024, 4000000 // (beams * vocab))))
        return dict(op=op, groups=groups, beams=beams, vocab=vocab, dtype=rng.choice(list(DTYPES)),
                    masked=rng.random() < 0.5, finished=rng.random() < 0.5, strided=rng.random() < 0.3)
    beams = rng.randint(1, 32)
    size = log_int(rng, 300, 90000)
    groups = log_int(rng, 1, max(1, min(2048, 90000000 // (beams * size))))
    return dict(op=op, groups=groups, beams=beams, size=size)


# -- inputs ---------------------------------------------------------------------------------

def padded_empty(rows, cols, dtype):
    """Rows on 16-byte boundaries, as the framework keeps 8-bit matrices."""
    return torch.empty((rows, -(-cols // 16) * 16), dtype=dtype, device='cuda')[:, :cols]


def values(gen, m, k):
    """Hidden-state like values: normal, with channels and rows of quite different size."""
    x = torch.randn((m, k), generator=gen, device='cuda')
    x *= torch.exp(0.7 * torch.randn((1, k), generator=gen, device='cuda'))
    x *= torch.exp(0.7 * torch.randn((m, 1), generator=gen, device='cuda'))
    return x


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    op = case['op']
    state = dict(case=case)
    if op == 'quantize':
        m, k, dtype = case['m'], case['k'], DTYPES[case['dtype']]
        x = values(gen, m, k).to(dtype)
        if case['strided']:
            wide = torch.zeros((m, k + 7), dtype=dtype, device='cuda')
            wide[:, 3:3 + k] = x
            x = wide[:, 3:3 + k]
        state.update(x=x)
    elif op == 'matmul':
        m, n, k = case['m'], case['n'], case['k']
        for name, rows, block in (('a', m, 1), ('w', n, BLOCK)):
            q, scale = plain_quantize(values(gen, rows, k) * (1.0 if name == 'a' else k ** -0.5), block)
            held = padded_empty(rows, k, torch.uint8)
            held.copy_(q.view(torch.uint8))
            state[name] = held.view(torch.float8_e4m3fn)
            state[name + '_scale'] = scale
        state.update(bias=None, add=None)
        if case['epilogue']:
            state['bias'] = torch.randn(n, generator=gen, device='cuda')
            state['add'] = torch.randn((m, n), generator=gen, device='cuda')
    elif op == 'select':
        g, w, v, dtype = case['groups'], case['beams'], case['vocab'], DTYPES[case['dtype']]
        x = 2.5 * torch.randn((g * w, v), generator=gen, device='cuda')
        x = x.to(dtype)
        if case['strided']:
            wide = torch.zeros((g * w, v + 5), dtype=dtype, device='cuda')
            wide[:, 1:1 + v] = x
            x = wide[:, 1:1 + v]
        scores = -20.0 * torch.rand((g, w), generator=gen, device='cuda')
        # A conversation's first step: one beam holds the prompt, the others nothing.
        first = torch.rand((g, 1), generator=gen, device='cuda') < 0.1
        later = torch.arange(w, device='cuda')[None, :] > 0
        scores = torch.where(first & later, -math.inf, scores)
        finished = allowed = None
        if case['finished']:
            finished = torch.rand((g, w), generator=gen, device='cuda') < 0.25
        if case['masked']:
            allowed = torch.ones(v, dtype=torch.bool, device='cuda')
            allowed[PAD:PAD + 2] = False
            allowed[torch.rand(v, generator=gen, device='cuda') < 0.02] = False
        state.update(logits=x, scores=scores, finished=finished, allowed=allowed)
    else:
        g, w, s = case['groups'], case['beams'], case['size']
        state['states'] = torch.randn((g * w, s), generator=gen, device='cuda')
        # Slots in order of score: the better a beam, the more of them follow it.
        u = torch.rand((g, w), generator=gen, device='cuda')
        state['parents'] = (u * u * w).to(torch.int32).clamp_(max=w - 1)
    return state


# -- plain forms ------------------------------------------------------------------------------

def plain_quantize(x, rows):
    m, k = x.shape
    mb, kb = -(-m // rows), -(-k // BLOCK)
    blocks = torch.zeros((mb * rows, kb * BLOCK), dtype=torch.float32, device=x.device)
    blocks[:m, :k] = x
    blocks = blocks.view(mb, rows, kb, BLOCK)
    amax = blocks.abs().amax((1, 3))
    scale = (amax / torch.full_like(amax, E4M3_MAX)).clamp(min=TINY)
    q = (blocks / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(mb * rows, kb * BLOCK)[:m, :k], scale


def dequantize(q, scale, rows, dtype):
    m, k = q.shape
    s = scale.to(dtype).repeat_interleave(rows, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]
    return q.to(dtype) * s


def plain_matmul(a, a_scale, w, w_scale, bias, add, dtype):
    y = dequantize(a, a_scale, 1, torch.float32) @ dequantize(w, w_scale, BLOCK, torch.float32).t()
    if bias is not None:
        y = y + bias
    if add is not None:
        y = y + ADD * add
    return y.to(dtype)


def plain_select(logits, scores, finished, allowed):
    g, w = scores.shape
    v = logits.shape[1]
    x = logits.double().view(g, w, v)
    if allowed is not None:
        x = torch.where(allowed, x, -math.inf)
    m = x.amax(2, keepdim=True)
    lse = m + (x - m).exp().sum(2, keepdim=True).log()
    total = scores.double()[:, :, None] + (x - lse)
    if finished is not None:
        same = torch.where(torch.arange(v, device=x.device) == PAD, scores.double()[:, :, None], -math.inf)
        total = torch.where(finished[:, :, None], same, total)
    total = torch.where(total.isfinite(), total, -math.inf).view(g, w * v)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :w], at[:, :w]
    none = best == -math.inf
    slot = torch.arange(w, device=x.device).expand(g, w)
    parents = torch.where(none, slot, at // v)
    tokens = torch.where(none, PAD, at % v)
    done = none | (tokens == END)
    if finished is not None:
        done = done | finished.gather(1, parents)
    return best.float(), tokens.to(torch.int32), parents.to(torch.int32), done


def plain_reorder(states, parents):
    g, w = parents.shape
    rows = (torch.arange(g, device=states.device)[:, None] * w + parents).view(-1)
    return states.copy_(states[rows])


def run(state):
    case = state['case']
    op = case['op']
    if own:
        blockscale, decoding = package()
        if op == 'quantize':
            return blockscale.quantize(state['x'], case['rows'])
        if op == 'matmul':
            return blockscale.matmul(state['a'], state['a_scale'], state['w'], state['w_scale'], state['bias'],
                                     state['add'], ADD, DTYPES[case['out']])
        if op == 'select':
            return decoding.beam_select(state['logits'], state['scores'], state['finished'], state['allowed'], END, PAD)
        return decoding.reorder(state['states'], state['parents'])
    if op == 'quantize':
        return plain_quantize(state['x'], case['rows'])
    if op == 'matmul':
        return plain_matmul(state['a'], state['a_scale'], state['w'], state['w_scale'], state['bias'], state['add'],
                            DTYPES[case['out']])
    if op == 'select':
        return plain_select(state['logits'], state['scores'], state['finished'], state['allowed'])
    return plain_reorder(state['states'], state['parents'])


def work(case):
    size = {'fp32': 4, 'bf16': 2, 'fp16': 2}
    if case['op'] == 'quantize':
        m, k = case['m'], case['k']
        scales = -(-m // case['rows']) * -(-k // BLOCK)
        return dict(bytes=m * k * (size[case['dtype']] + 1) + 4 * scales, flops=3 * m * k)
    if case['op'] == 'matmul':
        m, n, k = case['m'], case['n'], case['k']
        kb = -(-k // BLOCK)
        moved = (m + n) * k + 4 * kb * (m + -(-n // BLOCK)) + m * n * size[case['out']]
        if case['epilogue']:
            moved += 4 * n + 4 * m * n
        return dict(bytes=moved, flops=2 * m * n * k)
    if case['op'] == 'select':
        rows, v = case['groups'] * case['beams'], case['vocab']
        moved = rows * v * size[case['dtype']] + rows * (4 + 4 + 4 + 4 + 1)
        return dict(bytes=moved + (rows if case['finished'] else 0) + (v if case['masked'] else 0), flops=4 * rows * v)
    # Slots follow u^2 of the beams: the mean share of beams that some slot reads, and of slots that move.
    w, total = case['beams'], case['groups'] * case['beams'] * case['size'] * 4
    p = [math.sqrt((i + 1) / w) - math.sqrt(i / w) for i in range(w)]
    read = sum(1 - (1 - q) ** w for q in p) / w
    moves = 1 - sum(p) / w
    return dict(bytes=total * (read + moves) + 4 * case['groups'] * w, flops=0)


# -- the definition in 64 bits -----------------------------------------------------------------

def round_e4m3(v):
    """To the nearest e4m3 value (3 mantissa bits, smallest normal 2^-6, ties to even)."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'quantize':
        x, rows = state['x'].double(), case['rows']
        m, k = x.shape
        scale = torch.zeros((-(-m // rows), -(-k // BLOCK)), dtype=torch.float64, device='cuda')
        q = torch.empty_like(x)
        for j in range(scale.shape[1]):
            part = x[:, j * BLOCK:(j + 1) * BLOCK]
            top = part.abs().amax(1)
            if rows > 1:
                full = torch.zeros(scale.shape[0] * rows, dtype=torch.float64, device='cuda')
                full[:m] = top
                top = full.view(-1, rows).amax(1)
            scale[:, j] = (top / E4M3_MAX).clamp(min=TINY)
            by_row = scale[:, j].repeat_interleave(rows)[:m] if rows > 1 else scale[:, j]
            # The division that the 8-bit value rounds is by the scale as it is held, in 32 bits.
            held = by_row.float().double()
            q[:, j * BLOCK:(j + 1) * BLOCK] = round_e4m3((part / held[:, None]).float().double())
        return q, scale
    if case['op'] == 'matmul':
        m, n, k = case['m'], case['n'], case['k']
        y = torch.zeros((m, n), dtype=torch.float64, device='cuda')
        row_block = torch.arange(n, device='cuda') // BLOCK
        for j in range(state['a_scale'].shape[1]):
            at = slice(j * BLOCK, min(k, (j + 1) * BLOCK))
            part = state['a'][:, at].double() @ state['w'][:, at].double().t()
            part *= state['a_scale'][:, j].double()[:, None]
            part *= state['w_scale'][row_block, j].double()[None, :]
            y += part
        if case['epilogue']:
            y += state['bias'].double()
            y += ADD * state['add'].double()
        return y
    if case['op'] == 'select':
        g, w, v = case['groups'], case['beams'], case['vocab']
        best = torch.full((g, w), -math.inf, dtype=torch.float64)
        x, scores = state['logits'].double(), state['scores'].double().view(-1)
        if state['allowed'] is not None:
            x = x.masked_fill(~state['allowed'], -math.inf)
        logp = x - torch.logsumexp(x, 1, keepdim=True)
        logp += scores[:, None]
        if state['finished'] is not None:
            over = state['finished'].view(-1)
            logp[over] = -math.inf
            logp[over, PAD] = scores[over]
        best = torch.topk(logp.view(g, w * v), w, dim=1).values
        return best, None, None, None
    g, w = case['groups'], case['beams']
    old, parents = state['states'].double().view(g, w, -1), state['parents'].long()
    new = torch.empty_like(old)
    for j in range(w):
        new[:, j] = old[torch.arange(g, device='cuda'), parents[:, j]]
    return new.view(g * w, -1)
