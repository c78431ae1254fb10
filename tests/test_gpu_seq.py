"""Rotary positions, attention over packed sequences and attention over a paged cache (video_rep_learning_amd.ops) against their 64-bit
statements (oracle/seq.py), within bounds that follow from the kernels' roundings; then what a user can do with them: other strides,
padding, non-finite values where nobody looks, streams, graphs, and the four of them in a row."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import seq as OS  # noqa: E402
from video_rep_learning_amd import ops  # noqa: E402

DEV = 'cuda'
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ['fp32', 'bf16', 'fp16']


def randn(*shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def within(got, want, bound, what):
    err = (got.detach().double().cpu() - want).abs()
    over = err - bound
    assert not torch.isnan(err).any() and (over <= 0).all(), '%s: off by %.3e where %.3e is allowed (worst of %d)' % (
        what, err.flatten()[over.argmax()].item(), bound.flatten()[over.argmax()].item(), err.numel())


def cum(lengths, first=0):
    out = [first]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def cu_tensor(c):
    return torch.tensor(c, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ rotary
ROTARY = [  # tokens, hq, hk, d, sections, interleaved, pos dtype, far
    (1, 1, 1, 8, (4,), False, torch.int32, 0),
    (96, 8, 8, 32, (12, 4), False, torch.int64, 0),
    (77, 12, 3, 64, (8, 12, 12), False, torch.int64, 10 ** 6),
    (130, 5, 5, 40, (7, 6), True, torch.int32, 1000),
    (33, 4, 2, 128, (16, 24, 24), True, torch.int64, 10 ** 9),
    (19, 3, 1, 24, (5,), False, torch.float32, 0),
    (64, 2, 2, 80, (3, 1, 1), True, torch.float32, 3000),
    (5, 1, 1, 256, (100, 28), False, torch.int32, 7),
]


def positions(tokens, axes, dtype, far, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(-5, 900, (tokens, axes), generator=g)
    p[:, 0] += far
    return (p.float() + torch.rand(tokens, axes, generator=g) if dtype == torch.float32 else p.to(dtype)).to(DEV)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('t,hq,hk,d,sections,il,pdt,far', ROTARY)
def test_rotary_and_its_gradient(dtype, t, hq, hk, d, sections, il, pdt, far):
    qkv = randn(t, hq + 2 * hk, d, dtype=dtype, seed=1)
    q, k = qkv[:, :hq].requires_grad_(), qkv[:, hq:hq + hk].detach().requires_grad_()
    pos, freqs = positions(t, len(sections), pdt, far, 2), ops.rotary_freqs(sections)
    yq, yk = ops.rotary(q, k, pos, freqs, sections, interleaved=il)
    gq, gk = randn(t, hq, d, dtype=dtype, seed=3), randn(t, hk, d, dtype=dtype, seed=4)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for x, y, inv, what in ((q, yq, False, 'q'), (k, yk, False, 'k'), (gq, dq, True, 'dq'), (gk, dk, True, 'dk')):
        want = OS.rotate(x, pos, freqs, sections, il, inverse=inv)
        within(y, want, OS.rotate_bound(x, want, sections, il, dtype), what)
    only, none = ops.rotary(q.detach(), None, pos, freqs, sections, interleaved=il)
    assert none is None and torch.equal(only, yq)


def test_rotary_keeps_lengths_and_differences():
    """Against differences: rotation is linear, so y(x + e) - y(x) is the gradient's transpose applied to e up to two roundings of each."""
    t, h, d, sections = 20, 2, 16, (5, 3)
    q = randn(t, h, d, dtype=torch.float32, seed=5).requires_grad_()
    pos, freqs = positions(t, 2, torch.int64, 50, 6), ops.rotary_freqs(sections, base=500.0)
    w = randn(t, h, d, dtype=torch.float32, seed=7)
    y, _ = ops.rotary(q, None, pos, freqs, sections)
    dq, = torch.autograd.grad(y, q, w)
    e = randn(t, h, d, dtype=torch.float32, seed=8)
    with torch.no_grad():
        diff = ((ops.rotary(q + e, None, pos, freqs, sections)[0] - ops.rotary(q - e, None, pos, freqs, sections)[0]).double() * w.double()).sum() / 2
    lin = (dq.double() * e.double()).sum()
    mag = (w.double().abs() * (q.double().abs() + e.double().abs())).sum() * 4
    assert abs(diff - lin) <= 16 * OS.U32 * mag


def make_cache(pages, page, hk, d, dtype, seed):
    return randn(pages, page, hk, d, dtype=dtype, seed=seed), randn(pages, page, hk, d, dtype=dtype, seed=seed + 1)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('page,hq,hk,d,sections,il', [(16, 8, 8, 32, (12, 4), False), (7, 4, 2, 40, (20,), True), (1, 3, 1, 24, (3, 2, 1), False),
                                                      (64, 6, 2, 128, (16, 24, 24), True)])
def test_rotary_append_writes_its_slots_and_nothing_else(dtype, page, hq, hk, d, sections, il):
    news, olds = [3, 0, 1, 21, 2], [0, 4, 2 * page, 5, page - 1]
    width = max((a + b + page - 1) // page for a, b in zip(news, olds))
    pages = 5 * width + 2
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(3))[:5 * width].view(5, width).int().to(DEV)
    seq = [b for b, n in enumerate(news) for _ in range(n)] + [-1, 5, 2, 2, 0]                 # padding, no such stream,
    index = [o + i for n, o in zip(news, olds) for i in range(n)] + [0, 0, -1, width * page, 2 ** 31 - 1]   # no such index
    t = len(seq)
    table[4, 0] = pages                       # a page outside the cache, and a negative one
    table[4, width - 1] = -7
    kc, vc = make_cache(pages, page, hk, d, dtype, 11)
    want_k, want_v = kc.double().cpu(), vc.double().cpu()
    qkv = randn(t, hq + 2 * hk, d, dtype=dtype, seed=12)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    pos, freqs = positions(t, len(sections), torch.int64, 100, 13), ops.rotary_freqs(sections)
    qo = ops.rotary_append(q, k, v, pos, freqs, sections, kc, vc, table, torch.tensor(seq, dtype=torch.int32, device=DEV),
                           torch.tensor(index, dtype=torch.int32, device=DEV), interleaved=il)
    wq = OS.rotate(q, pos, freqs, sections, il)
    within(qo, wq, OS.rotate_bound(q, wq, sections, il, dtype), 'q')
    wk = OS.rotate(k, pos, freqs, sections, il)
    wb = OS.rotate_bound(k, wk, sections, il, dtype)
    bound = torch.zeros_like(want_k)
    for i, (b, j) in enumerate(zip(seq, index)):
        if 0 <= b < 5 and 0 <= j < width * page:
            pg = int(table[b, j // page])
            if 0 <= pg < pages:
                want_k[pg, j % page], want_v[pg, j % page], bound[pg, j % page] = wk[i], v[i].double().cpu(), wb[i]
    within(kc, want_k, bound, 'k cache')
    assert torch.equal(vc.double().cpu(), want_v)


# ------------------------------------------------------------------------------------------------ packed attention
LENGTHS = {
    'one': [1],
    'short': [1, 0, 2, 31, 32, 33, 0, 5],
    'edges': [63, 64, 65, 127, 129],
    'long': [300, 1, 517],
    'many': [3] * 70,
    'swarm': [2, 0, 1, 3] * 150,                        # more than the sequences that get tiles of their own
    'far': [1100, 3],                                   # few rows that walk far: eight waves share a tile's keys
    'pairs': [2600, 35],                                # with many heads: two waves for each 32 rows of a wide tile
    'wide': [300, 1, 0, 33, 129, 64, 517, 31] * 4,      # with 16 heads: enough rows for the form whose workgroups own 128
}
PACKED = [  # lengths, hq, hk, d, frame
    ('one', 1, 1, 8, 1), ('one', 4, 2, 64, 0),
    ('short', 8, 8, 32, 3), ('short', 4, 1, 40, 1), ('short', 3, 3, 96, 0),
    ('edges', 2, 2, 64, 1), ('edges', 6, 2, 128, 1), ('edges', 2, 1, 80, 7),
    ('long', 2, 2, 32, 6), ('long', 3, 1, 64, 0), ('long', 2, 2, 128, 100000),
    ('many', 2, 2, 16, 1), ('many', 5, 5, 48, 2),
    ('swarm', 2, 1, 32, 1), ('swarm', 2, 2, 64, 0),
    ('far', 2, 1, 64, 1), ('far', 1, 1, 32, 0), ('far', 2, 2, 24, 5), ('far', 4, 1, 128, 1),
    ('wide', 16, 16, 32, 1), ('wide', 16, 16, 64, 0), ('wide', 32, 16, 80, 3), ('wide', 16, 16, 128, 1), ('wide', 18, 9, 24, 0),
    ('pairs', 16, 8, 128, 1), ('pairs', 16, 8, 104, 5), ('pairs', 24, 24, 64, 1),
]


def run_packed(q, k, v, cu, frame, do, scale=None):
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out = ops.packed_attention(q, k, v, cu, frame=frame, scale=scale)
    return (out,) + torch.autograd.grad(out, (q, k, v), do)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('lengths,hq,hk,d,frame', PACKED)
def test_packed_attention_and_its_gradients(dtype, lengths, hq, hk, d, frame):
    c = cum(LENGTHS[lengths])
    t = c[-1]
    q, k, v = (randn(t, h, d, dtype=dtype, seed=20 + i, scale=s) for i, (h, s) in enumerate(((hq, 1.5), (hk, 1.0), (hk, 1.0))))
    do = randn(t, hq, d, dtype=dtype, seed=24)
    got = run_packed(q, k, v, cu_tensor(c), frame, do)
    want = OS.packed(q, k, v, c, frame, do=do)
    for x, nm in zip(got, ('out', 'dq', 'dk', 'dv')):
        assert x.dtype == dtype
        within(x, want[nm], want[nm + '_b'], nm)
    with torch.no_grad():
        assert torch.equal(ops.packed_attention(q, k, v, cu_tensor(c), frame=frame), got[0])       # the same without statistics


@pytest.mark.parametrize('dtype', DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize('lengths,h,d,frame', [([2, 2, 3, 1, 2], 1, 40, 1), ([2] * 20, 3, 80, 0), ([31, 5, 128, 2, 64], 2, 64, 1), ([4] * 30, 2, 128, 3),
                                               ([100, 3, 20] * 8, 2, 96, 1), ([40, 2, 9] * 40, 12, 64, 1), ([30, 3, 128] * 20, 16, 32, 0)],
                         ids=['pairs', 'couples', 'split', 'fours', 'split 96', 'wide', 'wide 32'])
def test_gradients_of_short_sequences_keep_their_bits(dtype, lengths, h, d, frame):
    """What is left of dP - delta in short sequences is small beside both: delta must not come from the rounded output alone, and dS must
    not lose what 16 bits take."""
    c = cum(lengths)
    q, k, v = (randn(c[-1], h, d, dtype=dtype, seed=390 + i, scale=s) for i, s in enumerate((1.5, 1.0, 1.0)))
    do = randn(c[-1], h, d, dtype=dtype, seed=394)
    got = run_packed(q, k, v, cu_tensor(c), frame, do)
    want = OS.packed(q, k, v, c, frame, do=do, fine=True)
    for x, nm in zip(got, ('out', 'dq', 'dk', 'dv')):
        within(x, want[nm], want[nm + '_b'], nm)


@pytest.mark.parametrize('lengths,h,d,frame,small', [([2000, 30], 2, 64, 1, 8), ([1500], 3, 32, 0, 10), ([400, 700] * 6, 8, 64, 0, 8),
                                                     ([2600, 45], 16, 128, 1, 6), ([40, 3], 2, 64, 1, 12)], ids=['split', 'all keys', 'wide', 'pairs', 'short'])
def test_fp16_gradients_far_below_one(lengths, h, d, frame, small):
    """Output gradients of 2^-6 to 2^-12: dS lies where fp16 has few bits or none, the gradients themselves do not."""
    c, dtype = cum(lengths), torch.float16
    q, k, v = (randn(c[-1], h, d, dtype=dtype, seed=395 + i) for i in range(3))
    do = randn(c[-1], h, d, dtype=dtype, seed=399, scale=2.0 ** -small)
    got = run_packed(q, k, v, cu_tensor(c), frame, do)
    for x, nm in zip(got[1:], ('dq', 'dk', 'dv')):
        x = x[:, -1:]
        y = OS.packed(q[:, -1:], k[:, -1:], v[:, -1:], c, frame, do=do[:, -1:])[nm]
        # roundings of the operand, of the result and of the output that delta reads, none above 2^-11, random in sign; elements below
        # 2^-14 round to steps of 2^-24
        error = (x.double().cpu() - y).norm()
        assert error <= 3 * 2.0 ** -11 / math.sqrt(3) * y.norm() + 2.0 ** -25 * math.sqrt(y.numel()), (nm, error / y.norm())


@pytest.mark.parametrize('dtype,lengths,hq,hk,d,frame', [
    (torch.bfloat16, [6000, 70], 8, 4, 64, 1),       # 408 workgroups of 128 rows: all on the card at once, two rounds there and back
    (torch.bfloat16, [2600, 45], 12, 4, 96, 1),      # 288: the second round is a part of one
    (torch.float16, [4200, 130], 15, 5, 80, 6),      # 555, all heads' tiles in turn
    (torch.float32, [5200], 3, 1, 32, 1),            # the split form, eight waves a tile
    (torch.bfloat16, [6500], 8, 2, 128, 0),          # walks of the whole sequence, two waves in turn only where causal
    (torch.bfloat16, [6500], 8, 2, 128, 1)], ids=['there and back', 'part of a round', 'heads in turn', 'split', 'all keys', 'pairs'])
def test_long_sequences(dtype, lengths, hq, hk, d, frame):
    """Thousands of tokens, one group of heads of them compared."""
    c, g, at = cum(lengths), hq // hk, hk - 1
    q, k, v, do = (randn(c[-1], h, d, dtype=dtype, seed=380 + i) for i, h in enumerate((hq, hk, hk, hq)))
    got = run_packed(q, k, v, cu_tensor(c), frame, do)
    hs, ks = slice(at * g, at * g + g), slice(at, at + 1)
    want = OS.packed(q[:, hs], k[:, ks], v[:, ks], c, frame, do=do[:, hs])
    for x, nm in zip(got, ('out', 'dq', 'dk', 'dv')):
        within(x[:, hs if nm in ('out', 'dq') else ks], want[nm], want[nm + '_b'], nm)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('frame,behind,hq,hk', [(0, 61, 4, 2), (1, 61, 4, 2), (4, 61, 4, 2), (1, 4100, 16, 16)])
def test_packed_attention_leaves_rows_of_no_sequence_alone(dtype, frame, behind, hq, hk):
    """Rows before the first and behind the last sequence hold NaN (uninitialised padding): zeros out, zero gradients, and the rows of
    sequences come out as if the others were not there."""
    c = cum([40, 0, 75], first=3)
    t, d = c[-1] + behind, 64
    q, k, v, do = (randn(t, h, d, dtype=dtype, seed=30 + i) for i, h in enumerate((hq, hk, hk, hq)))
    for x in (q, k, v, do):
        x[:3] = math.nan
        x[c[-1]:] = math.nan
    got = run_packed(q, k, v, cu_tensor(c), frame, do)
    inner = slice(3, c[-1])
    alone = run_packed(q[inner], k[inner], v[inner], cu_tensor([x - 3 for x in c]), frame, do[inner])
    want = OS.packed(*(x[inner] for x in (q, k, v)), [x - 3 for x in c], frame, do=do[inner])
    for x, y, nm in zip(got, alone, ('out', 'dq', 'dk', 'dv')):
        assert (x[:3] == 0).all() and (x[c[-1]:] == 0).all(), nm
        within(x[inner], want[nm], want[nm + '_b'], nm)
        within(y, want[nm], want[nm + '_b'], nm)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
def test_packed_attention_hides_what_a_row_does_not_see(dtype, bad):
    """Non-finite keys and values of one token: the rows that see it change, no other row does -- not the earlier ones of the same tile,
    not the next sequence's."""
    c, hq, hk, d, at = cum([50, 70, 20]), 2, 1, 32, 50 + 37
    t = c[-1]
    q, k, v = (randn(t, h, d, dtype=dtype, seed=40 + i) for i, h in enumerate((hq, hk, hk)))
    clean = OS.packed(q, k, v, c, 1)
    sees = torch.zeros(t, dtype=torch.bool)
    sees[at:c[2]] = True
    v2 = v.clone()
    v2[at, :, 5] = bad
    out = ops.packed_attention(q, k, v2, cu_tensor(c), frame=1)
    within(out[~sees], clean['out'][~sees], clean['out_b'][~sees], 'unseen value')
    other = [i for i in range(d) if i != 5]
    within(out[sees][..., other], clean['out'][sees][..., other], clean['out_b'][sees][..., other], 'other channels')
    got = out[sees][..., 5].double().cpu()
    assert torch.isnan(got).all() if math.isnan(bad) else (got == bad).all()
    k2 = k.clone()
    k2[at] = bad
    out = ops.packed_attention(q, k2, v, cu_tensor(c), frame=1)
    within(out[~sees], clean['out'][~sees], clean['out_b'][~sees], 'unseen key')
    # two infinities of different sign meet
    v2[at + 3, :, 5] = -bad
    out = ops.packed_attention(q, k, v2, cu_tensor(c), frame=1)
    assert torch.isnan(out[at + 3:c[2], :, 5]).all() and (math.isnan(bad) or not torch.isnan(out[at:at + 3, :, 5]).any())


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('lengths,hq,hk', [([45, 30, 90], 4, 2), ([450, 35] + [100] * 37, 16, 16), ([1600, 35], 2, 1)],
                         ids=['split', 'wide', 'far'])
def test_packed_attention_gradients_hide_other_sequences(dtype, lengths, hq, hk):
    """A sequence whose inputs or output gradients are not finite leaves its neighbours' gradients as they are."""
    c, d = cum(lengths), 64
    t = c[-1]
    q, k, v, do = (randn(t, h, d, dtype=dtype, seed=50 + i) for i, h in enumerate((hq, hk, hk, hq)))
    want = OS.packed(q, k, v, c, 1, do=do)
    keep = torch.ones(t, dtype=torch.bool)
    keep[c[1]:c[2]] = False
    for which in range(4):
        xs = [x.clone() for x in (q, k, v, do)]
        xs[which][c[1] + 4] = math.nan
        xs[which][c[1] + 9] = math.inf
        got = run_packed(xs[0], xs[1], xs[2], cu_tensor(c), 1, xs[3])
        for x, nm in zip(got, ('out', 'dq', 'dk', 'dv')):
            within(x[keep], want[nm][keep], want[nm + '_b'][keep], '%s with a bad %s' % (nm, 'qkvd'[which]))
        # causal: what comes before the bad token inside its own sequence
        within(got[0][c[1]:c[1] + 4], want['out'][c[1]:c[1] + 4], want['out_b'][c[1]:c[1] + 4], 'earlier rows')


@pytest.mark.parametrize('dtype,hq,hk,d', [(torch.bfloat16, 16, 8, 128), (torch.float16, 16, 8, 120), (torch.float32, 24, 24, 64)], ids=IDS[1:] + IDS[:1])
def test_packed_attention_gradients_hide_other_sequences_from_pairs_of_waves(dtype, hq, hk, d):
    """As above, where two waves share a row tile: each redoes its own half of the tiles."""
    c = cum([2600, 45])
    q, k, v, do = (randn(c[-1], h, d, dtype=dtype, seed=55 + i) for i, h in enumerate((hq, hk, hk, hq)))
    want = OS.packed(q, k, v, c, 1, do=do)
    for which in range(4):
        xs = [x.clone() for x in (q, k, v, do)]
        xs[which][c[1] + 4] = math.nan
        xs[which][c[1] - 3, :, 5] = math.inf             # the last rows of the long one: no earlier row's output or dQ sees them
        got = run_packed(xs[0], xs[1], xs[2], cu_tensor(c), 1, xs[3])
        for x, nm in zip(got[:2], ('out', 'dq')):
            within(x[:c[1] - 3], want[nm][:c[1] - 3], want[nm + '_b'][:c[1] - 3], '%s with a bad %s' % (nm, 'qkvd'[which]))
        for x, nm in zip(got[:2], ('out', 'dq')):
            within(x[c[1]:c[1] + 4], want[nm][c[1]:c[1] + 4], want[nm + '_b'][c[1]:c[1] + 4], '%s of the next sequence' % nm)


@pytest.mark.parametrize('lengths,hq,hk,d,dtypes', [([500, 450, 500], 12, 6, 64, DTYPES), ([450, 35] + [100] * 37, 8, 4, 64, DTYPES),
                                                    ([2600, 45], 16, 8, 128, DTYPES[1:2]), ([2600, 45], 16, 8, 120, DTYPES[2:]),
                                                    ([2600, 45], 16, 16, 64, DTYPES[:1])],
                         ids=['split, two heads a workgroup', 'wide, two heads a workgroup', 'pairs bf16', 'pairs fp16', 'pairs fp32'])
def test_key_gradients_past_a_bad_query(lengths, hq, hk, d, dtypes):
    """A query or output gradient that is not finite early in a long sequence: the keys behind it, some of them in its own tile, are not
    seen by it and keep their gradients, which their waves take again over their whole walk; an output gradient with one infinite
    channel leaves the other channels of every dV as they are."""
    c, at = cum(lengths), 100
    for dtype in dtypes:
        q, k, v, do = (randn(c[-1], h, d, dtype=dtype, seed=350 + i) for i, h in enumerate((hq, hk, hk, hq)))
        want = OS.packed(q, k, v, c, 1, do=do)
        rows, keys = torch.arange(c[-1]) != at, torch.arange(c[-1]) > at
        other = [i for i in range(d) if i != 5]
        for which, bad in (('q', math.nan), ('q', math.inf), ('do', math.nan), ('do', -math.inf)):
            q2, do2 = q.clone(), do.clone()
            if which == 'q':
                q2[at] = bad
            else:
                do2[at, :, 5] = bad
            got = run_packed(q2, k, v, cu_tensor(c), 1, do2)
            for x, nm, keep in zip(got, ('out', 'dq', 'dk', 'dv'), (rows, rows, keys, keys)):
                within(x[keep], want[nm][keep], want[nm + '_b'][keep], '%s behind a bad %s' % (nm, which))
            if which == 'do':
                within(got[0], want['out'], want['out_b'], 'out')
                within(got[3][..., other], want['dv'][..., other], want['dv_b'][..., other], 'the other channels of dv')


def test_packed_attention_gradient_against_differences():
    """Central differences of the fp32 forward: f = sum w * out.  The forward is off by its bounds, so f by b = sum |w| bound, the quotient
    by b / h; the step's own error is h^2 / 6 of the third derivative, taken from halving the step."""
    c, hq, hk, d, frame = cum([17, 1, 30]), 2, 1, 16, 3
    t = c[-1]
    x = [randn(t, h, d, dtype=torch.float32, seed=60 + i, scale=0.7) for i, h in enumerate((hq, hk, hk))]
    w = randn(t, hq, d, dtype=torch.float32, seed=64)
    grads = run_packed(*x, cu_tensor(c), frame, w)[1:]
    bound = (w.double().abs().cpu() * OS.packed(*x, c, frame)['out_b']).sum().item()

    def f(xs):
        return (ops.packed_attention(*xs, cu_tensor(c), frame=frame).double() * w.double()).sum().item()
    for i in range(3):
        e = randn(*x[i].shape, dtype=torch.float32, seed=70 + i)
        quotient = []
        for h in (2.0 ** -4, 2.0 ** -5):
            quotient.append((f([y + h * e if j == i else y for j, y in enumerate(x)]) - f([y - h * e if j == i else y for j, y in enumerate(x)])) / (2 * h))
        lin = (grads[i].double() * e.double()).sum().item()
        # x +- h e rounds too: one step of 32 bits of x, carried by the gradient
        rounding = (grads[i].double().abs() * x[i].double().abs()).sum().item() * 4 * OS.U32 * 2.0 ** 5
        assert abs(quotient[1] - lin) <= abs(quotient[0] - quotient[1]) + 2 * bound * 2.0 ** 5 + rounding, (i, quotient, lin)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_packed_attention_other_strides(dtype):
    """Slices of a fused projection, heads before tokens, an odd start (copied), channels not contiguous (copied), broadcast keys."""
    c, hq, hk, d = cum([33, 60]), 4, 2, 32
    t = c[-1]
    q, k, v, do = (randn(t, h, d, dtype=dtype, seed=80 + i) for i, h in enumerate((hq, hk, hk, hq)))
    base = run_packed(q, k, v, cu_tensor(c), 1, do)
    fused = torch.cat([q, k, v], 1)
    tr = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    odd = [torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape) for x in (q, k, v)]
    last = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    for xs in ((fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:]), tr, odd, last):
        got = run_packed(*xs, cu_tensor(c).long(), 1, do.transpose(0, 1).contiguous().transpose(0, 1))
        assert all(torch.equal(a, b) for a, b in zip(base, got))
    # one key head for all, broadcast by the caller: the gradient of the broadcast input is the sum of the heads'
    one = randn(t, 1, d, dtype=torch.float32, seed=90).requires_grad_()
    qf, vf, dof = q.float(), v.float(), do.float()
    out = ops.packed_attention(qf, one.expand(t, hk, d), vf, cu_tensor(c), frame=1)
    g, = torch.autograd.grad(out, one, dof)
    want = OS.packed(qf, one.detach().expand(t, hk, d), vf, c, 1, do=dof)
    within(g[:, 0], want['dk'].sum(1), want['dk_b'].sum(1) + OS.U32 * want['dk'].abs().sum(1), 'broadcast key')


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('t,h,d', [(1, 8, 32), (5, 1, 32), (1, 1, 8)])
def test_one_token_or_one_head_in_any_memory_order(dtype, t, h, d):
    """A dimension of size 1 may have any stride (channels first, narrow slices): the same bits as from a tensor of its own."""
    qkv = [randn(t, h, d, dtype=dtype, seed=95 + i) for i in range(3)]
    pos, freqs, cu = positions(t, 1, torch.int64, 3, 98), ops.rotary_freqs((d // 2,)), cu_tensor([0, t])
    table, n = torch.tensor([[1, 0, 2]], dtype=torch.int32, device=DEV), torch.tensor([t], device=DEV)
    seq, index = torch.zeros(t, dtype=torch.int32, device=DEV), torch.arange(t, dtype=torch.int32, device=DEV)

    def all_of_them(q, k, v):
        q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
        a, b = ops.rotary(q, k, pos, freqs, (d // 2,))
        got = [a, b, *torch.autograd.grad((a, b), (q, k), (v, q))]
        got += run_packed(q, k, v, cu, 1, v.detach())
        with torch.no_grad():
            kc, vc = make_cache(3, 2, h, d, dtype, 99)
            got += [ops.rotary_append(q, k, v, pos, freqs, (d // 2,), kc, vc, table, seq, index), kc, vc]
            got += [ops.paged_attention(q[None], kc, vc, table, n), ops.paged_attention(q[:, None], kc, vc, table.expand(t, 3), n.expand(t))]
        return got
    want = all_of_them(*qkv)
    for order in ((2, 0, 1), (0, 2, 1), (1, 2, 0)):
        xs = [x.permute(order).contiguous().permute([order.index(i) for i in range(3)]) for x in qkv]
        assert all(torch.equal(a, b) for a, b in zip(want, all_of_them(*xs)))
    xs = [torch.cat([x, x[..., :4]], 2)[..., :d] for x in qkv]
    assert all(torch.equal(a, b) for a, b in zip(want, all_of_them(*xs)))


RISING = [('short', 4, 2, 40, 1), ('edges', 2, 1, 80, 0), ('long', 3, 1, 64, 5), ('far', 2, 1, 64, 1), ('far', 1, 1, 32, 0), ('wide', 16, 16, 32, 1),
          ('wide', 16, 8, 128, 0), ('swarm', 2, 1, 32, 1), ('pairs', 16, 8, 128, 1), ('pairs', 16, 16, 64, 1)]


def rising(x, lengths, height, seed):
    """Keys whose products with rising_queries() climb by `height` over each sequence."""
    u = torch.randn(x.shape[-1], generator=torch.Generator().manual_seed(seed)).sign().to(DEV)
    step = torch.cat([torch.arange(n) / max(n, 1) for n in lengths]).to(DEV)
    return (x.float() * 0.7 + step[:, None, None] * height / x.shape[-1] * u).to(x.dtype), u


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('scale', [0.6, 0.03], ids=['large scale', 'small scale'])
@pytest.mark.parametrize('lengths,hq,hk,d,frame', RISING)
def test_packed_attention_with_scores_that_rise_along_the_keys(dtype, scale, lengths, hq, hk, d, frame):
    """A scale of the caller's, and scores that climb by 60 over a sequence: most rows take a new maximum again and again, in every form."""
    lens = LENGTHS[lengths]
    c = cum(lens)
    q, k, v = (randn(c[-1], h, d, dtype=dtype, seed=360 + i) for i, h in enumerate((hq, hk, hk)))
    k, u = rising(k, lens, 60 / scale, 364)
    q = (q.float() * 0.3 + u).to(dtype)
    do = randn(c[-1], hq, d, dtype=dtype, seed=365)
    got = run_packed(q, k, v, cu_tensor(c), frame, do, scale=scale)
    want = OS.packed(q, k, v, c, frame, scale=scale, do=do)
    for x, nm in zip(got, ('out', 'dq', 'dk', 'dv')):
        within(x, want[nm], want[nm + '_b'], nm)


@pytest.mark.parametrize('scale', [1e-39, 3e-38, 1e-20])
def test_scales_that_leave_no_difference_between_scores(scale):
    """Every visible key weighs the same, in each form."""
    for lengths, hq in ((LENGTHS['short'], 2), (LENGTHS['far'], 2), (LENGTHS['wide'], 16), ([2600, 35], 16)):
        c, d = cum(lengths), 64
        q, k, v = (randn(c[-1], hq, d, dtype=torch.float32, seed=310 + i) for i in range(3))
        out = ops.packed_attention(q, k, v, cu_tensor(c), frame=1, scale=scale)
        want = OS.packed(q[:, :1], k[:, :1], v[:, :1], c, 1, scale=scale)
        within(out[:, :1], want['out'], want['out_b'], 'out of %d heads' % hq)
    for lengths in ([99, 0, 1], [5000]):
        q, kc, vc, table, lens = make_paged(lengths, 1, 16, 2, 2, 64, torch.float32, 315)
        want, bound = OS.paged(q, kc, vc, table, lens, 1, scale=scale)
        within(ops.paged_attention(q, kc, vc, table, lens, scale=scale), want, bound, 'paged')


def first_of_all(s, limits):
    """The key of each row's largest score among those it sees, and whether it stands out by more than 32 bits round: a sum of up to 128
    products is off by at most 24 steps of the magnitudes' sum, which is some five times the largest score."""
    s = s.masked_fill(torch.arange(s.shape[1])[None] >= torch.as_tensor(limits)[:, None], -math.inf)
    top = s.topk(min(2, s.shape[1]), 1)
    clear = torch.ones(s.shape[0], dtype=torch.bool)
    if s.shape[1] > 1:
        clear = top.values[:, 0] - top.values[:, 1] > 2.0 ** -16 * s.masked_fill(s.isinf(), 0).abs().amax(1)
        assert clear.sum() >= 0.98 * len(clear) - 1
    return top.indices[:, 0], clear


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('lengths,hq,d', [([40, 1, 35], 2, 32), ([350, 70], 2, 64), ([40, 30, 9] * 28, 16, 64), ([1300], 16, 128)],
                         ids=['split', 'far', 'wide', 'pairs'])
def test_scores_far_beyond_the_range_of_exponents(dtype, lengths, hq, d):
    """Scores of 10^9 (fp16) to 10^21: each row takes the value of its largest score's key, exactly."""
    c, big, d = cum(lengths), 1.5e4 if dtype == torch.float16 else 1e10, 64 if len(lengths) == 1 and dtype == torch.float32 else d
    q, k = (randn(c[-1], hq, d, dtype=torch.float32, seed=320 + i).mul_(big).clamp_(-6e4 if big < 1e5 else -1e12, 6e4 if big < 1e5 else 1e12).to(dtype)
            for i in range(2))
    v = randn(c[-1], hq, d, dtype=dtype, seed=322)
    out = ops.packed_attention(q, k, v, cu_tensor(c), frame=1, scale=1.0)
    for h in (0, hq - 1):
        for a, b in zip(c[:-1], c[1:]):
            at, clear = first_of_all(q[a:b, h].double().cpu() @ k[a:b, h].double().cpu().t(), range(1, b - a + 1))
            assert torch.equal(out[a:b, h].cpu()[clear], v[a:b, h].cpu()[at[clear]]), (h, a)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('lengths,width', [([99, 1, 0, 40], 0), ([2500, 3], 300)])
def test_paged_scores_far_beyond_the_range_of_exponents(dtype, lengths, width):
    big = 1.5e4 if dtype == torch.float16 else 1e10
    q, kc, vc, table, lens = make_paged(lengths, 2, 16, 2, 1, 64, dtype, 330)
    table = torch.cat([table, torch.full((len(lengths), width), -1, dtype=torch.int32, device=DEV)], 1)
    q, kc = ((x.float() * big).clamp(-6e4 if big < 1e5 else -1e12, 6e4 if big < 1e5 else 1e12).to(dtype) for x in (q / 1.5, kc))
    out = ops.paged_attention(q, kc, vc, table, lens, scale=1.0)
    for b, n in enumerate(lengths):
        pages = table[b, :-(-n // 16)].long()
        k, v = (x[pages].flatten(0, 1)[:n, 0].cpu() for x in (kc, vc))
        for i in range(2):
            for h in range(2):
                if n - 2 + i < 0:
                    assert (out[b, i, h] == 0).all()
                    continue
                at, clear = first_of_all((q[b, i, h].double().cpu() @ k.double().t())[None], [n - 1 + i])
                assert not clear or torch.equal(out[b, i, h].cpu(), v[at[0]]), (b, i, h)


@pytest.mark.parametrize('dtype', DTYPES[:2], ids=IDS[:2])
def test_a_key_of_the_lowest_values(dtype):
    """A key filled with the type's lowest value has a score of some 10^36: all of the weight, or none of it, by the sign of the query's sum."""
    n, d = 90, 32
    q, k, v = (randn(n, 1, d, dtype=dtype, seed=340 + i, scale=s) for i, s in enumerate((1e-3, 1.0, 1.0)))
    k[0] = torch.finfo(dtype).min
    out = ops.packed_attention(q, k, v, cu_tensor([0, n]), frame=1)
    first = q[:, 0].double().sum(1).cpu() < 0
    first[0] = True                                                # it sees nothing else
    assert torch.equal(out[:, 0].cpu()[first], v[0].cpu().expand(n, d)[first])
    rest = OS.attend(q[1:, 0], k[1:, 0], v[1:, 0], range(1, n), d ** -0.5, dtype)
    within(out[1:, 0].cpu()[~first[1:]], rest['out'][~first[1:]], rest['out_b'][~first[1:]], 'without it')


def test_packed_attention_nothing_to_do():
    z = torch.zeros(0, 2, 32, device=DEV).requires_grad_()
    out = ops.packed_attention(z, z, z, cu_tensor([0, 0]), frame=1)
    out.sum().backward()
    assert out.shape == (0, 2, 32) and z.grad.shape == (0, 2, 32)
    q = randn(9, 2, 32, dtype=torch.float32, seed=1).requires_grad_()
    out = ops.packed_attention(q, q, q, cu_tensor([0, 0, 0]), frame=0)         # rows, but no sequence holds them
    out.sum().backward()
    assert (out == 0).all() and (q.grad == 0).all()
    y, _ = ops.rotary(z.detach(), None, torch.zeros(0, 1, dtype=torch.int64, device=DEV), ops.rotary_freqs((16,)), (16,))
    assert y.shape == (0, 2, 32)


def test_packed_attention_survives_bounds_out_of_order():
    """Bounds that do not ascend or leave the rows give no meaningful rows, but nothing outside the operands is touched."""
    q = randn(200, 2, 32, dtype=torch.bfloat16, seed=2).requires_grad_()
    for c in ([50, 10, 300], [-40, 20, 10 ** 9], [200, 0, 200], [0, 2 ** 31 - 1, -2 ** 31]):
        out = ops.packed_attention(q, q, q, cu_tensor(c), frame=3)
        torch.autograd.grad(out, q, torch.ones_like(out))
    torch.cuda.synchronize()


def test_packed_attention_far_rows():
    """Token strides that put the last rows behind 2^31 elements."""
    t, h, d = 130, 1, 64
    stride = (1 << 31) // 100 // 8 * 8
    buf = torch.empty(stride * (t - 1) + 3 * d, device=DEV, dtype=torch.bfloat16)
    q, k, v = (buf[i * d:].as_strided((t, h, d), (stride, d, 1)) for i in range(3))
    dense = [randn(t, h, d, dtype=torch.bfloat16, seed=100 + i) for i in range(3)]
    for x, y in zip((q, k, v), dense):
        x.copy_(y)
    cu = cu_tensor([0, 60, t])
    assert torch.equal(ops.packed_attention(q, k, v, cu, frame=1), ops.packed_attention(*dense, cu, frame=1))


# ------------------------------------------------------------------------------------------------ paged attention
PAGED = [  # lengths, new, page, hq, hk, d, frame
    ([1], 1, 16, 1, 1, 8, 1),
    ([99], 3, 16, 8, 8, 32, 3),
    ([0, 1, 2, 31, 32, 33, 64, 65], 1, 7, 4, 2, 40, 1),
    ([5, 0, 130, 2], 3, 1, 6, 2, 64, 1),
    ([700, 3, 257], 2, 24, 8, 1, 128, 0),
    ([1300, 2600, 1], 1, 64, 16, 4, 128, 1),
    ([90, 4], 6, 16, 16, 2, 96, 6),
    ([4, 200], 5, 16, 40, 2, 80, 1),            # 100 rows of one key head: several tiles
    ([3000], 1, 128, 2, 2, 64, 1),
    ([0] * 66 + [2500] + [0] * 3 + [1, 40, 900] * 20 + [0] * 9, 1, 16, 4, 2, 32, 1),           # 139 streams, many of them empty
    ([700, 0, 1400] + [130, 5] * 31, 2, 24, 8, 4, 40, 0),                                       # 65 streams, four key heads each
    ([4100, 300], 9, 64, 8, 2, 64, 1),          # 36 rows of one key head, long
]


def make_paged(lengths, new, page, hq, hk, d, dtype, seed, spare=2):
    """Streams whose pages lie in a random order in a cache that holds NaN wherever no stream's key is."""
    need = [-(-n // page) for n in lengths]
    pages, width = sum(need) + spare, max(max(need), 1) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    kc, vc = make_cache(pages, page, hk, d, dtype, seed)
    used = torch.zeros(pages, page, dtype=torch.bool)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for j in range(need[b]):
            pg = order.pop()
            table[b, j] = pg
            used[pg, :min(page, n - j * page)] = True
    kc[~used.to(DEV)] = math.nan
    vc[~used.to(DEV)] = math.nan
    q = randn(len(lengths), new, hq, d, dtype=dtype, seed=seed + 5, scale=1.5)
    return q, kc, vc, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('lengths,new,page,hq,hk,d,frame', PAGED)
def test_paged_attention(dtype, lengths, new, page, hq, hk, d, frame):
    q, kc, vc, table, lens = make_paged(lengths, new, page, hq, hk, d, dtype, 110)
    out = ops.paged_attention(q, kc, vc, table, lens, frame=frame)
    want, bound = OS.paged(q, kc, vc, table, lens, frame)
    within(out, want, bound, 'out')
    wide = torch.cat([table, torch.full((len(lengths), 700), -1, dtype=torch.int32, device=DEV)], 1)     # room for much longer streams
    within(ops.paged_attention(q, kc, vc, wide, lens.long(), frame=frame), want, bound, 'wide table')
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.paged_attention(qt, kc, vc, table, lens, frame=frame), out)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('scale', [0.6, 0.03], ids=['large scale', 'small scale'])
@pytest.mark.parametrize('lengths,new,page,hq,hk,d,frame', [PAGED[i] for i in (1, 3, 5, 7, 8, 10, 11)])
def test_paged_attention_with_scores_that_rise_along_the_keys(dtype, scale, lengths, new, page, hq, hk, d, frame):
    q, kc, vc, table, lens = make_paged(lengths, new, page, hq, hk, d, dtype, 370)
    for b, n in enumerate(lengths):
        for j in range(-(-n // page)):
            m, pg = min(page, n - j * page), int(table[b, j])
            u = torch.randn(d, generator=torch.Generator().manual_seed(371)).sign().to(DEV)
            step = (torch.arange(j * page, j * page + m, device=DEV) / n)[:, None, None]
            kc[pg, :m] = (kc[pg, :m].float() * 0.7 + step * (60 / scale / d) * u).to(dtype)
    q = (q.float() * 0.2 + torch.randn(d, generator=torch.Generator().manual_seed(371)).sign().to(DEV)).to(dtype)
    want, bound = OS.paged(q, kc, vc, table, lens, frame, scale=scale, low=True)
    within(ops.paged_attention(q, kc, vc, table, lens, frame=frame, scale=scale), want, bound, 'out')


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_paged_attention_bad_pages_and_lengths(dtype):
    """Pages outside the cache hold no keys; a length beyond the table's pages is cut to them, a negative one is 0."""
    q, kc, vc, table, _ = make_paged([200, 200, 64, 64], 1, 16, 4, 2, 32, dtype, 120)
    table[0, 3] = kc.shape[0]
    table[0, 7] = -5
    table[1, :] = 2 ** 31 - 1
    lens = torch.tensor([200, 200, -3, 10 ** 9], dtype=torch.int32, device=DEV)
    out = ops.paged_attention(q, kc, vc, table, lens, frame=1)
    want, bound = OS.paged(q, kc, vc, table, lens, 1)
    within(out, want, bound, 'out')
    assert (out[1] == 0).all() and (out[2] == 0).all()


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_paged_attention_hides_later_new_tokens(dtype):
    """Of several new tokens the earlier ones do not see the later ones' keys, whatever these hold."""
    q, kc, vc, table, lens = make_paged([67], 3, 16, 2, 2, 32, dtype, 130)
    want, bound = OS.paged(q, kc, vc, table, lens, 1)
    pg, row = int(table[0, 66 // 16]), 66 % 16
    kc[pg, row], vc[pg, row] = math.nan, math.inf
    out = ops.paged_attention(q, kc, vc, table, lens, frame=1)
    within(out[:, :2], want[:, :2], bound[:, :2], 'earlier tokens')
    assert torch.isnan(out[:, 2]).all()


@pytest.mark.parametrize('dtype', DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize('lengths,new,page,hq,hk,d,frame', [PAGED[2], PAGED[4], PAGED[5], PAGED[6], PAGED[7], PAGED[11]])
def test_paged_attention_rounds_once(dtype, lengths, new, page, hq, hk, d, frame):
    """16-bit results are the one rounding of a 32-bit sum: the weights lose no bits that count on the way into their product."""
    q, kc, vc, table, lens = make_paged(lengths, new, page, hq, hk, d, dtype, 110)
    want, bound = OS.paged(q, kc, vc, table, lens, frame, low=True)
    within(ops.paged_attention(q, kc, vc, table, lens, frame=frame), want, bound, 'out')


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('bad', [math.inf, -math.inf])
@pytest.mark.parametrize('length,width', [(97, 0), (3000, 0)])
def test_paged_attention_carries_infinite_values(dtype, bad, length, width):
    """An infinite value among the visible ones is that row's result in its channel, in the middle of a walk as beside masked places."""
    for at in (40, length - 1):
        q, kc, vc, table, lens = make_paged([length], 2, 16, 4, 2, 32, dtype, 135)
        want, bound = OS.paged(q, kc, vc, table, lens, 1)
        # weights of this key in all rows, far from what 16 bits flush
        pg, row = int(table[0, at // 16]), at % 16
        vc[pg, row, :, 5] = bad
        out = ops.paged_attention(q, kc, vc, table, lens, frame=1)
        sees = [i for i in range(2) if at < length - 1 + i]
        assert (out[0, sees][..., 5] == bad).all()
        other = [i for i in range(32) if i != 5]
        within(out[..., other], want[..., other], bound[..., other], 'other channels')


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('n', [20, 90, 300])
def test_value_gradients_carry_infinite_output_gradients(dtype, n):
    q, k, v, do = (randn(n, 2, 32, dtype=dtype, seed=400 + i, scale=0.5) for i in range(4))
    do[n // 2, :, 5] = math.inf
    got = run_packed(q, k, v, cu_tensor([0, n]), 1, do)
    assert (got[3][:n // 2 + 1, :, 5] == math.inf).all() and torch.isfinite(got[3][n // 2 + 1:]).all()


def test_paged_attention_far_pages():
    """Pages behind 2^31 elements of the cache, written by rotary_append and read back."""
    page, hk, d = 64, 8, 128
    pages = (1 << 31) // (page * hk * d) + 5
    kc, vc = (torch.empty(pages, page, hk, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    n = 150
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device=DEV)
    q, k, v = (randn(n, hk, d, dtype=torch.bfloat16, seed=140 + i) for i in range(3))
    pos, freqs = torch.arange(n, device=DEV)[:, None].contiguous(), ops.rotary_freqs((64,))
    seq, index = torch.zeros(n, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    turned = ops.rotary_append(q, k, v, pos, freqs, (64,), kc, vc, table, seq, index)
    out = ops.paged_attention(turned[-1:][None], kc, vc, table, torch.tensor([n], device=DEV), frame=1)
    tq, tk = ops.rotary(q, k, pos, freqs, (64,))
    assert torch.equal(tq, turned)
    want = OS.packed(tq, tk, v, [0, n], 1)
    within(out[0, 0], want['out'][-1], want['out_b'][-1], 'far pages')


# ------------------------------------------------------------------------------------------------ the four of them in a row
def project(x, w, hq, hk, d):
    qkv = (x.float() @ w).to(x.dtype).view(x.shape[0], hq + 2 * hk, d)
    return qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('ntok,page,hq,hk', [(3, 16, 8, 8), (1, 7, 4, 2)])
def test_streaming_equals_the_whole_video(dtype, ntok, page, hq, hk):
    """Two layers of attention, causal by frame, over three videos of different lengths at once (rotary + packed_attention) and frame by
    frame over a paged cache (rotary_append + paged_attention): the second layer reads the first one's outputs, so both sides' bounds are
    carried through one layer by the reference run on the first side's own first-layer output."""
    d, sections, frames = 32, (12, 4), [9, 30, 1]
    lengths = [f * ntok for f in frames]
    c, t = cum(lengths), sum(lengths)
    x = randn(t, hq * d, dtype=dtype, seed=150)
    w = [randn(hq * d, (hq + 2 * hk) * d, dtype=torch.float32, seed=151 + i, scale=(hq * d) ** -0.5) for i in range(2)]
    step = torch.cat([torch.arange(n) for n in lengths]).to(DEV)
    pos = torch.stack([step // ntok, step % ntok], 1).contiguous()
    freqs = ops.rotary_freqs(sections)
    cu = cu_tensor(c)
    whole, y, inputs = [], x, []
    for i in range(2):
        q, k, v = project(y, w[i], hq, hk, d)
        q, k = ops.rotary(q, k, pos, freqs, sections)
        inputs.append((q, k, v))
        y = ops.packed_attention(q, k, v, cu, frame=ntok).view(t, hq * d)
        whole.append(y)
    width = -(-max(lengths) // page)
    caches = [make_cache(3 * width, page, hk, d, dtype, 160 + 2 * i) for i in range(2)]
    table = torch.randperm(3 * width, generator=torch.Generator().manual_seed(5)).view(3, width).int().to(DEV)
    got = torch.zeros_like(x)
    for f in range(max(frames)):
        live = [b for b in range(3) if f < frames[b]]
        rows = torch.tensor([c[b] + f * ntok + j for b in live for j in range(ntok)], device=DEV)
        seq = torch.tensor([b for b in live for _ in range(ntok)], dtype=torch.int32, device=DEV)
        index = step[rows].int()
        lens = torch.full((len(live),), (f + 1) * ntok, dtype=torch.int32, device=DEV)
        y = x[rows]
        for i in range(2):
            # the second layer starts from the whole run's first layer, so that the two sides differ by one layer's roundings
            q, k, v = project(y if i == 0 else whole[0][rows], w[i], hq, hk, d)
            q = ops.rotary_append(q, k, v, pos[rows], freqs, sections, *caches[i], table, seq, index)
            out = ops.paged_attention(q.view(len(live), ntok, hq, d), *caches[i], table[live], lens, frame=ntok)
            y = out.view(len(rows), hq * d)
            if i == 0:
                first = OS.packed(*inputs[0], c, ntok) if f == 0 else first
                within(y.view(-1, hq, d), first['out'][rows.cpu()], 2 * first['out_b'][rows.cpu()] + 1e-6, 'first layer, frame %d' % f)
        got[rows] = y
    second = OS.packed(*inputs[1], c, ntok)
    within(got.view(t, hq, d), second['out'], 2 * second['out_b'] + 1e-6, 'second layer')


def test_training_through_rotary_and_attention():
    """Gradients of a projection, rotary positions and attention in a row, against the same composition in 64 bits by autograd."""
    hq, hk, d, sections, c = 4, 2, 32, (10, 6), cum([30, 7, 51])
    t = c[-1]
    x = randn(t, 64, dtype=torch.float32, seed=170)
    w = randn(64, (hq + 2 * hk) * d, dtype=torch.float32, seed=171, scale=0.1).requires_grad_()
    pos, freqs = positions(t, 2, torch.int64, 9, 172), ops.rotary_freqs(sections)
    wo = randn(t, hq, d, dtype=torch.float32, seed=173)
    q, k, v = project(x, w, hq, hk, d)
    q, k = ops.rotary(q, k, pos, freqs, sections)
    out = ops.packed_attention(q, k, v, cu_tensor(c), frame=3)
    g, = torch.autograd.grad(out, w, wo)

    w64 = w.detach().double().cpu().requires_grad_()
    qkv = (x.double().cpu() @ w64).view(t, hq + 2 * hk, d)
    ang = torch.cat([pos.cpu()[:, a:a + 1].double() * freqs.cpu()[s:s + m] for a, (s, m) in enumerate(((0, 10), (10, 6)))], 1)[:, None]

    def turn(z):
        a, b = z[..., :16], z[..., 16:]
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    q64, k64, v64, loss = turn(qkv[:, :hq]), turn(qkv[:, hq:hq + hk]), qkv[:, hq + hk:], 0
    for a, b in zip(c[:-1], c[1:]):
        i = torch.arange(b - a)
        mask = i[None] < (i[:, None] // 3 + 1) * 3
        for h in range(hq):
            s = (q64[a:b, h] @ k64[a:b, h // 2].t() * d ** -0.5).masked_fill(~mask, -math.inf)
            loss = loss + ((s.softmax(1) @ v64[a:b, h // 2]) * wo[a:b, h].double().cpu()).sum()
    g64, = torch.autograd.grad(loss, w64)
    # every element is a sum over t rows of 32-bit quantities that carry some hundred roundings each (projection 64, score 32, softmax,
    # products over the sequence): 2^-24 * 512 of the largest gradient
    assert (g.double().cpu() - g64).abs().max().item() <= 512 * OS.U32 * g64.abs().max().item()


# ------------------------------------------------------------------------------------------------ streams, graphs, repetition
def test_a_second_derivative_is_refused():
    q, k, v, do = (randn(40, 2, 32, dtype=torch.float32, seed=300 + i).requires_grad_() for i in range(4))
    out = ops.packed_attention(q, k, v, cu_tensor([0, 40]), frame=1)
    dq, = torch.autograd.grad(out, q, do, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), q)
    turned, _ = ops.rotary(q, k, torch.arange(40, device=DEV)[:, None].contiguous(), ops.rotary_freqs((16,)), (16,))
    dq, = torch.autograd.grad(turned, q, do, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), do)


def test_append_ignores_slots_outside_32_bits_and_one_cache_for_both():
    kc, vc = make_cache(4, 16, 2, 32, torch.float32, 310)
    before = kc.clone()
    q = randn(3, 2, 32, dtype=torch.float32, seed=311)
    pos, freqs = torch.zeros(3, 1, dtype=torch.int64, device=DEV), ops.rotary_freqs((16,))
    table = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device=DEV)
    seq = torch.tensor([0, 2 ** 32, 0], device=DEV)
    index = torch.tensor([2 ** 32 + 5, 9, -2 ** 32 + 1], device=DEV)
    ops.rotary_append(q, q, q, pos, freqs, (16,), kc, vc, table, seq, index)
    assert torch.equal(kc, before)
    with pytest.raises(ValueError):
        ops.rotary_append(q, q, q, pos, freqs, (16,), kc, kc, table, seq, index)


def test_same_bits_every_time():
    c = cum([700, 3, 1000])
    t = c[-1]
    q, k, v, do = (randn(t, h, 64, dtype=torch.bfloat16, seed=180 + i) for i, h in enumerate((8, 2, 2, 8)))
    a, b = (run_packed(q, k, v, cu_tensor(c), 1, do) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    p = make_paged([5000, 300], 1, 16, 8, 2, 64, torch.bfloat16, 190)
    assert torch.equal(ops.paged_attention(*p, frame=1), ops.paged_attention(*p, frame=1))


def test_another_stream():
    p = make_paged([3000, 70], 1, 16, 8, 2, 64, torch.float32, 200)
    want = ops.paged_attention(*p, frame=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [ops.paged_attention(*p, frame=1) for _ in range(3)]
    outs.append(ops.paged_attention(*p, frame=1))              # at the same time on the default stream: workspaces of their own
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(want, o) for o in outs)


def test_graphs_replay_on_new_inputs():
    """A streaming step (rotary_append + paged_attention) and a training step (forward and gradients) captured into two graphs, replayed in
    turn with new inputs, new lengths and eager work between; each replay equals the eager result."""
    hq, hk, d, page, B = 8, 2, 64, 16, 3
    freqs, sections = ops.rotary_freqs((20, 12)), (20, 12)
    kc, vc = make_cache(200, page, hk, d, torch.bfloat16, 210)
    table = torch.randperm(200, generator=torch.Generator().manual_seed(1))[:180].view(3, 60).int().to(DEV)
    qkv = torch.zeros(B, hq + 2 * hk, d, device=DEV, dtype=torch.bfloat16)
    pos, index = torch.zeros(B, 2, dtype=torch.int64, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    seq, lens = torch.arange(B, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)

    def serve():
        q = ops.rotary_append(qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:], pos, freqs, sections, kc, vc, table, seq, index)
        return ops.paged_attention(q[:, None], kc, vc, table, lens, frame=1)
    t = 150
    xs = [torch.zeros(t, h, d, device=DEV, dtype=torch.float16).requires_grad_() for h in (hq, hk, hk)]
    do, cu = torch.zeros(t, hq, d, device=DEV, dtype=torch.float16), cu_tensor([0, 1, 2])

    def learn():
        out = ops.packed_attention(*xs, cu, frame=1)
        return (out.detach(),) + torch.autograd.grad(out, xs, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        serve()
    with torch.cuda.stream(side):
        learn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1), torch.no_grad():
        served = serve()
    with torch.cuda.graph(g2):
        learned = learn()
    for i in range(4):
        qkv.copy_(randn(B, hq + 2 * hk, d, dtype=torch.bfloat16, seed=220 + i))
        index.copy_(torch.tensor([i, 200 * i, 900 - i], dtype=torch.int32))
        pos.copy_(torch.stack([index.long() * 3, index.long()], 1))
        lens.copy_(index + 1)
        with torch.no_grad():
            for x, h in zip(xs, (hq, hk, hk)):
                x.copy_(randn(t, h, d, dtype=torch.float16, seed=230 + 7 * i + h))
        do.copy_(randn(t, hq, d, dtype=torch.float16, seed=250 + i))
        cu.copy_(torch.tensor([0, 20 * i + 1, t - i], dtype=torch.int32))
        g1.replay()
        g2.replay()
        a, b = served.clone(), [x.clone() for x in learned]
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(a, serve())
        assert all(torch.equal(x, y) for x, y in zip(b, learn()))
