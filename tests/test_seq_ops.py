"""What the operators of token sequences refuse, checked without a GPU: argument checks of ops come before any launch, and so do those of the
C entry points (their pointers are never read here)."""
import ctypes

import pytest
import torch

from video_rep_learning_amd import _lib, ops

P = 4096            # an aligned address that nothing reads


@pytest.fixture(scope='module')
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from video_rep_learning_amd.csrc import build
        build.build()
    return _lib.load()


def heads(t=4, h=2, d=32, dtype=torch.float32):
    return torch.zeros(t, h, d, dtype=dtype)


def test_cpu_tensors_are_refused():
    q, pos = heads(), torch.zeros(4, 1, dtype=torch.int64)
    freqs = ops.rotary_freqs((16,), device='cpu')
    cache, table, i = torch.zeros(2, 4, 2, 32), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(_lib.MvfError):
        ops.rotary(q, q, pos, freqs, (16,))
    with pytest.raises(_lib.MvfError):
        ops.rotary_append(q, q, q, pos, freqs, (16,), cache, cache, table, i, i)
    with pytest.raises(_lib.MvfError):
        ops.packed_attention(q, q, q, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(_lib.MvfError):
        ops.paged_attention(q[None], cache, cache, table, torch.tensor([3]))


@pytest.mark.parametrize('q,k', [(heads(d=12), heads(d=12)), (heads(h=3), heads(t=5)), (heads(), heads(d=64)), (torch.zeros(4, 32), heads()),
                                 (heads(h=0), heads()), (heads(d=136), heads(d=136)[:3])])
def test_shapes_are_refused(q, k):
    with pytest.raises(ValueError):
        ops.packed_attention(q, k, k, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.rotary(q, k, torch.zeros(q.shape[0], 1, dtype=torch.int64), ops.rotary_freqs((4,), device='cpu'), (4,))


def test_paged_shapes_are_refused():
    for q in (torch.zeros(1, 32), torch.zeros(1, 1, 2, 36), torch.zeros(1, 1, 2, 136), torch.zeros(1, 0, 2, 32)):
        with pytest.raises(ValueError):
            ops.paged_attention(q, torch.zeros(2, 4, 2, 32), torch.zeros(2, 4, 2, 32), torch.zeros(1, 2, dtype=torch.int32), torch.tensor([3]))


@pytest.mark.parametrize('frame', [-1, 1.0, True, None, 2 ** 31])
def test_frame_argument(frame):
    with pytest.raises(ValueError):
        ops._frame_arg(frame)


@pytest.mark.parametrize('scale', [0.0, -1.0, float('nan'), float('inf')])
def test_scale_argument(scale):
    with pytest.raises(ValueError):
        ops._scale_arg(scale, 64)


@pytest.mark.parametrize('sections', [(), (0, 4), (-1,), (17,), (8, 8, 8), (1, 1, 1, 1)])
def test_sections_argument(sections):
    q = heads()
    with pytest.raises(ValueError):
        ops._rotary_args(torch.zeros(4, len(sections), dtype=torch.int64), torch.zeros(max(1, sum(sections)), dtype=torch.float64), sections, 4, 32, q)


def test_positions_and_freqs_arguments():
    q, f = heads(), ops.rotary_freqs((8, 8), device='cpu')
    assert f.dtype == torch.float64 and f[0] == 1 and f[8] == 1
    good = torch.zeros(4, 2, dtype=torch.int64)
    for pos, freqs in ((good.double(), f), (good[:, :1], f), (good[:3], f), (good, f.float()), (good, f[:15])):
        with pytest.raises(ValueError):
            ops._rotary_args(pos, freqs, (8, 8), 4, 32, q)


def test_cache_arguments():
    q = heads()
    ok = torch.zeros(2, 4, 2, 32)
    ops._cache_args(q, ok, ok.clone())
    for kc, vc in ((ok[0], ok), (ok, ok[:1]), (torch.zeros(2, 4, 3, 32),) * 2, (torch.zeros(2, 4, 2, 64),) * 2, (torch.zeros(0, 4, 2, 32),) * 2,
                   (ok.transpose(1, 2).contiguous().transpose(1, 2), ok)):
        with pytest.raises(ValueError):
            ops._cache_args(q, kc, vc)


def test_aligned_copies_only_what_it_must():
    x = torch.zeros(6, 4, 32)
    assert ops._aligned(x) is x and ops._aligned(x[:, 1:3]).data_ptr() == x[:, 1:3].data_ptr()
    for y in (x.transpose(1, 2), torch.zeros(6 * 4 * 32 + 1)[1:].view(6, 4, 32), x[:, :1].expand(6, 4, 32), torch.zeros(6, 4, 34)[..., :32]):
        z = ops._aligned(y)
        assert z.data_ptr() != y.data_ptr() and z.data_ptr() % 16 == 0 and z.is_contiguous() and torch.equal(z, y)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_aligned_gives_dimensions_of_size_one_strides_of_their_own(dtype):
    """torch calls these contiguous whatever stride the dimension of size 1 has: one token held channels first, one head, a narrow slice."""
    for y in (torch.randn(8, 32, 1).to(dtype).permute(2, 0, 1), torch.randn(4, 32, 1).to(dtype).transpose(1, 2),
              torch.randn(1, 1, 12 if dtype != torch.float32 else 10).to(dtype)[..., :8], torch.randn(1, 1, 8).to(dtype).expand(1, 1, 8),
              torch.randn(1, 8, 32, 1).to(dtype).permute(0, 3, 1, 2), torch.randn(2, 5, 16, 1).to(dtype).transpose(2, 3)):
        z = ops._aligned(y)
        a = 16 // y.element_size()
        assert torch.equal(z, y) and z.data_ptr() % 16 == 0 and z.stride(-1) == 1 and all(s > 0 and s % a == 0 for s in z.stride()[:-1])


@pytest.fixture
def on_cpu(monkeypatch):
    """The operators' Python side on CPU tensors: no device check; a launch leaves its results as they were allocated."""
    monkeypatch.setattr(ops, '_seq_operands', lambda first, *others: ops._SEQ_DT[first.dtype])
    return monkeypatch


def calls(grad):
    q, k, v = (torch.randn(4, 2, 32, requires_grad=grad) for _ in range(3))
    pos, freqs, cu = torch.zeros(4, 1, dtype=torch.int64), ops.rotary_freqs((16,), device='cpu'), torch.tensor([0, 4], dtype=torch.int32)
    kc, vc, table, i = torch.zeros(2, 4, 2, 32), torch.zeros(2, 4, 2, 32), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    return (q, k, v), {
        'rotary': lambda q, k, v: ops.rotary(q, k, pos, freqs, (16,))[0],
        'rotary, keys': lambda q, k, v: ops.rotary(q.detach(), k, pos, freqs, (16,))[1],
        'packed_attention': lambda q, k, v: ops.packed_attention(q, k, v, cu),
        'rotary_append': lambda q, k, v: ops.rotary_append(q, k, v, pos, freqs, (16,), kc, vc, table, i, i),
        'paged_attention': lambda q, k, v: ops.paged_attention(q[None], kc, vc, table, cu[1:])}


@pytest.mark.parametrize('which', range(3))
def test_forward_mode_derivatives_are_refused(on_cpu, which):
    """A dual operand has no requires_grad; its tangent must not be dropped without a word."""
    on_cpu.setattr(ops, '_launch', lambda *a: None)
    xs, fns = calls(False)
    for name, fn in fns.items():
        if name == 'rotary' and which != 0 or name == 'rotary, keys' and which != 1 or name == 'paged_attention' and which != 0:
            continue
        for mode in (True, False):
            with torch.set_grad_enabled(mode), torch.autograd.forward_ad.dual_level():
                dual = [torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)) if i == which else x for i, x in enumerate(xs)]
                with pytest.raises((NotImplementedError, ValueError)):
                    fn(*dual)
                fn(*xs)                                 # an open level alone changes nothing


@pytest.mark.filterwarnings('ignore::torch.jit.TracerWarning')
@pytest.mark.parametrize('name', ['rotary', 'rotary, keys', 'packed_attention', 'rotary_append', 'paged_attention'])
def test_tracing_is_refused(on_cpu, name):
    """A trace would hold the allocation of the results only."""
    from torch.fx.experimental.proxy_tensor import make_fx
    for grad in (False, True):
        xs, fns = calls(grad and not name.startswith(('rotary_append', 'paged')))
        with pytest.raises(_lib.MvfError):
            torch.jit.trace(fns[name], xs)
        with pytest.raises(_lib.MvfError):
            make_fx(fns[name])(*xs)


@pytest.mark.parametrize('which', [5, 6])
def test_append_refuses_caches_that_want_a_gradient(on_cpu, which):
    on_cpu.setattr(ops, '_launch', lambda *a: None)
    q, pos, i = heads(), torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)
    args = [q, q.clone(), q.clone(), pos, ops.rotary_freqs((16,), device='cpu'), torch.zeros(2, 4, 2, 32), torch.zeros(2, 4, 2, 32)]
    args[which].requires_grad_()
    rest = (torch.zeros(1, 2, dtype=torch.int32), i, i)
    with pytest.raises(ValueError, match='no gradient'):
        ops.rotary_append(*args[:5], (16,), *args[5:], *rest)
    with torch.no_grad():
        ops.rotary_append(*args[:5], (16,), *args[5:], *rest)


def test_append_tells_autograd_that_the_caches_changed(on_cpu):
    """A graph that saved a cache refuses to run backward over other values than it saw."""
    on_cpu.setattr(ops, '_launch', lambda *a: None)
    q, pos, i = heads(), torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)
    freqs, kc, vc = ops.rotary_freqs((16,), device='cpu'), torch.zeros(2, 4, 2, 32), torch.zeros(2, 4, 2, 32)
    for cache in (kc, vc):
        w = torch.ones(32, requires_grad=True)
        y = (cache * w).sum()
        with torch.no_grad():
            ops.rotary_append(q, q, q, pos, freqs, (16,), kc, vc, torch.zeros(1, 2, dtype=torch.int32), i, i)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.backward()


def test_rotary_refuses_angles_that_want_a_gradient(on_cpu):
    on_cpu.setattr(ops, '_launch', lambda *a: None)
    q, pos, freqs = heads(), torch.zeros(4, 1), ops.rotary_freqs((16,), device='cpu')
    for p, f in ((pos.clone().requires_grad_(), freqs), (pos, freqs.clone().requires_grad_())):
        for x in (q, q.clone().requires_grad_()):
            with pytest.raises(ValueError, match='no gradient'):
                ops.rotary(x, x, p, f, (16,))
        with torch.no_grad():
            ops.rotary(q, q, p, f, (16,))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match='no gradient'):
        ops.rotary(q, q, pos, torch.autograd.forward_ad.make_dual(freqs, torch.ones_like(freqs)), (16,))


def test_append_refuses_memory_that_it_would_read_and_write(on_cpu):
    on_cpu.setattr(ops, '_launch', lambda *a: None)
    pos, freqs, i = torch.zeros(4, 1, dtype=torch.int64), ops.rotary_freqs((16,), device='cpu'), torch.zeros(4, dtype=torch.int32)
    table, n = torch.zeros(1, 2, dtype=torch.int32), 2 * 4 * 2 * 32
    pool = torch.zeros(4 * n)

    def cache(at):
        return pool[at:at + n].view(2, 4, 2, 32)

    def rows(at):
        return pool[at:].as_strided((4, 2, 32), (64, 32, 1))

    def append(q, k, v, kc, vc):
        return ops.rotary_append(q, k, v, pos, freqs, (16,), kc, vc, table, i, i)
    x = torch.zeros(4, 2, 32)
    append(x, x, x, cache(0), cache(n))                                   # neighbours
    append(rows(2 * n), rows(2 * n), rows(2 * n + 256), cache(n), cache(0))
    for off in (0, 4, n // 2, n - 4):
        with pytest.raises(ValueError, match='share memory'):
            append(x, x, x, cache(off), cache(0))
        with pytest.raises(ValueError, match='share memory'):
            append(x, x, x, cache(0), cache(off))
    for bad in (rows(0), rows(2 * n - 64), rows(n + 64)):
        for at in range(3):
            with pytest.raises(ValueError, match='memory of a cache'):
                append(*(bad if j == at else x for j in range(3)), cache(0), cache(n))


FWD = dict(dtype=_lib.BF16, q=P, ldq=64, hsq=32, k=P, ldk=64, hsk=32, v=P, ldv=64, hsv=32, cu=P, n=1, out=P, stat=None, T=4, Hq=2, Hk=2, D=32,
           frame=1, scale=1.0)
BAD_ATTN = [('dtype', 2), ('q', None), ('q', P + 8), ('k', None), ('v', None), ('cu', None), ('out', None), ('out', P + 4), ('ldq', 0), ('ldq', 63),
            ('hsk', -32), ('ldv', 4), ('n', 0), ('T', 0), ('T', -1), ('Hq', 3), ('Hk', 0), ('frame', -1), ('scale', 0.0), ('scale', float('nan')),
            ('scale', float('inf'))]


@pytest.mark.parametrize('name,value', BAD_ATTN)
def test_packed_entry_points_refuse(lib, name, value):
    a = dict(FWD, **{name: value})
    assert lib.mvf_packed_attn_fwd(*a.values(), None) == 10001
    head = [a[n] for n in ('dtype', 'q', 'ldq', 'hsq', 'k', 'ldk', 'hsk', 'v', 'ldv', 'hsv', 'cu', 'n', 'out')]
    tail = [a[n] for n in ('T', 'Hq', 'Hk', 'D', 'frame', 'scale')]
    assert lib.mvf_packed_attn_bwd(*head, P, P, P, 1 << 40, P, P, P, *tail, None) == 10001


def test_packed_entry_points_with_rest_refuse_what_the_others_do(lib):
    def fwd(rest=P, **kw):
        a = dict(FWD, **kw)
        v = list(a.values())
        at = list(a).index('out') + 1
        return lib.mvf_packed_attn_fwd_rest(*v[:at], rest, *v[at:], None)

    def bwd(rest=P, d_out=P, ws=1 << 40, **kw):
        a = dict(FWD, **kw)
        head = [a[n] for n in ('dtype', 'q', 'ldq', 'hsq', 'k', 'ldk', 'hsk', 'v', 'ldv', 'hsv', 'cu', 'n', 'out')]
        return lib.mvf_packed_attn_bwd_rest(*head, rest, d_out, P, P, ws, P, P, P, *(a[n] for n in ('T', 'Hq', 'Hk', 'D', 'frame', 'scale')), None)
    for name, value in BAD_ATTN:
        assert fwd(**{name: value}) == 10001 and bwd(**{name: value}) == 10001, name
    assert fwd(rest=P + 8) == 10001 and bwd(rest=P + 8) == 10001 and bwd(d_out=None) == 10001 and bwd(ws=8) == 10001


@pytest.mark.parametrize('d', [0, 12, 136, -8])
def test_head_sizes_are_declined(lib, d):
    assert lib.mvf_packed_attn_fwd(*dict(FWD, D=d).values(), None) == 10002
    assert lib.mvf_paged_attn(_lib.F32, P, 64, 64, 32, P, P, P, P, P, None, 0, 1, 1, 2, 2, d, 1, 16, 1, 1, 1.0, None) == 10002


@pytest.mark.parametrize('missing', range(6))
def test_packed_backward_refuses_missing_buffers(lib, missing):
    bufs = [P] * 6
    bufs[missing] = None
    head = [FWD[n] for n in ('dtype', 'q', 'ldq', 'hsq', 'k', 'ldk', 'hsk', 'v', 'ldv', 'hsv', 'cu', 'n', 'out')]
    assert lib.mvf_packed_attn_bwd(*head, *bufs[:3], 1 << 40, *bufs[3:], 4, 2, 2, 32, 1, 1.0, None) == 10001


def test_packed_backward_workspace_is_asked_for_and_checked(lib):
    head = [FWD[n] for n in ('dtype', 'q', 'ldq', 'hsq', 'k', 'ldk', 'hsk', 'v', 'ldv', 'hsv', 'cu', 'n', 'out')]
    size = lib.mvf_packed_attn_bwd_workspace_bytes(_lib.BF16, 4, 1, 2, 2, 32)
    assert size >= 4 * 2 * 4                                                         # delta
    assert lib.mvf_packed_attn_bwd(*head, P, P, P, size - 1, P, P, P, 4, 2, 2, 32, 1, 1.0, None) == 10001
    # few key heads: the group's heads are shared out and their sums kept in fp32; many: they are not
    assert lib.mvf_packed_attn_bwd_workspace_bytes(_lib.BF16, 512, 1, 16, 4, 128) == 4 * (16 * 512 + 2 * 4 * 512 * 4 * 128)
    assert lib.mvf_packed_attn_bwd_workspace_bytes(_lib.BF16, 1 << 17, 1, 16, 4, 128) == 4 * 16 * (1 << 17)
    assert lib.mvf_packed_attn_bwd_workspace_bytes(_lib.BF16, 512, 1, 3, 2, 128) == 0


ROT = dict(dtype=_lib.F32, q=P, ldq=64, hsq=32, k=P, ldk=64, hsk=32, pos=P, pos_type=0, freqs=P, s0=8, s1=4, s2=0, il=0, inv=0, qo=P, ko=P, T=4,
           Hq=2, Hk=2, D=32)


@pytest.mark.parametrize('name,value', [('dtype', 2), ('q', None), ('k', None), ('pos', None), ('pos_type', 3), ('freqs', None), ('s0', 0), ('s1', 9),
                                        ('s2', -1), ('qo', None), ('ko', None), ('qo', P + 2), ('T', 0), ('Hq', 0), ('Hk', -1), ('ldq', 65),
                                        ('hsk', 0), ('D', 0), ('D', 8192)])
def test_rotary_entry_point_refuses(lib, name, value):
    assert lib.mvf_rotary(*dict(ROT, **{name: value}).values(), None) == 10001


def test_rotary_axes_have_to_follow_each_other(lib):
    assert lib.mvf_rotary(*dict(ROT, s1=0, s2=4).values(), None) == 10001
    assert lib.mvf_rotary(*dict(ROT, D=36).values(), None) == 10002


def test_append_entry_point_refuses(lib):
    ok = dict(dtype=_lib.F32, q=P, ldq=64, hsq=32, k=P, ldk=64, hsk=32, v=P, ldv=64, hsv=32, pos=P, pos_type=0, freqs=P, s0=8, s1=4, s2=0, il=0,
              qo=P, kc=P, vc=P, table=P, width=2, n_seqs=1, seq=P, index=P, n_pages=4, page=16, T=4, Hq=2, Hk=2, D=32)
    for name, value in (('v', None), ('v', P + 1), ('ldv', 3), ('qo', None), ('kc', None), ('vc', P + 8), ('table', None), ('width', 0), ('n_seqs', 0),
                        ('seq', None), ('index', None), ('n_pages', 0), ('page', 0), ('Hk', 0), ('T', 0)):
        assert lib.mvf_rotary_append(*dict(ok, **{name: value}).values(), None) == 10001, name


PAGED = dict(dtype=_lib.F32, q=P, qb=64, qn=64, qh=32, kc=P, vc=P, table=P, lens=P, out=P, ws=P, ws_bytes=1 << 30, B=1, n=1, Hq=2, Hk=2, D=32,
             n_pages=4, page=16, width=2, frame=1, scale=1.0)


@pytest.mark.parametrize('name,value', [('dtype', 7), ('q', None), ('q', P + 4), ('kc', None), ('vc', P + 2), ('table', None), ('lens', None),
                                        ('out', None), ('B', 0), ('n', 0), ('Hq', 3), ('Hk', 0), ('n_pages', 0), ('page', 0), ('width', 0),
                                        ('frame', -2), ('scale', 0.0), ('qb', 2), ('width', 2 ** 28)])
def test_paged_entry_point_refuses(lib, name, value):
    assert lib.mvf_paged_attn(*dict(PAGED, **{name: value}).values(), None) == 10001


def test_paged_workspace_is_asked_for_and_checked(lib):
    size = lib.mvf_paged_attn_workspace_bytes(1, 1, 2, 2, 32, 4096, 16)
    assert size > 0 and size % 4 == 0
    long = dict(PAGED, width=4096)
    assert lib.mvf_paged_attn(*dict(long, ws=None).values(), None) == 10001
    assert lib.mvf_paged_attn(*dict(long, ws_bytes=size - 1).values(), None) == 10001
    assert lib.mvf_paged_attn_workspace_bytes(1, 1, 3, 2, 32, 4096, 16) == 0
    assert lib.mvf_paged_attn_workspace_bytes(64, 1, 8, 8, 128, 1, 16) == 0          # one page per stream: nothing to join
    assert isinstance(ctypes.c_size_t(size).value, int)


def test_indices_outside_32_bits_stay_outside():
    """int64 indices are not cut to their low bits: 2^32 + 3 is not slot 3."""
    q = heads()
    got = ops._index_operand(torch.tensor([2 ** 32 + 3, -2 ** 40, 7, -1]), q, (4,), 'index')
    assert got.dtype == torch.int32 and got.tolist() == [2 ** 31 - 1, -2 ** 31, 7, -1]
    i32 = torch.tensor([1, 2], dtype=torch.int32)
    assert ops._index_operand(i32, q, (2,), 'seq') is i32


def test_sizes_beyond_the_kernels_counters_are_refused():
    far = torch.zeros(1, dtype=torch.bfloat16).expand(2 ** 30, 1, 8)
    with pytest.raises(ValueError):
        ops._heads(far, 'q')
    ops._heads(far[1:], 'q')
    with pytest.raises(ValueError):
        ops.packed_attention(far, far, far, torch.tensor([0, 4], dtype=torch.int32))


def test_paged_entry_point_refuses_more_keys_than_it_counts(lib):
    assert lib.mvf_paged_attn(*dict(PAGED, width=2 ** 21, page=1024).values(), None) == 10001
