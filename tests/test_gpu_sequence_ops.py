"""GPU: the sequence operators (rotary_embed, attn_window, window_cache_append, attn_window_step) against float64 forms
(oracle/sequence_oracle.py, which also derives the bounds used here)."""
import pytest
import torch

from helpers import ROOT  # noqa: F401  (puts the repository's root in sys.path)
from oracle import sequence_oracle as ref

from tempenslearnagg_qcnet_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _cu(lens):
    return torch.tensor([0] + torch.tensor(lens, dtype=torch.int64).cumsum(0).tolist())


def _check(got, r, dtype, dim, v, what=''):
    o, mag, reach, count = r
    got = got.cpu().double()
    assert got.shape == o.shape
    assert bool(torch.isfinite(got).all()), what
    tol = ref.tolerance(dtype, dim, o, mag, reach, count, float(v.double().abs().max()) if v.numel() else 0.0)
    ratio = ((got - o).abs() / tol)
    assert o.numel() == 0 or float(ratio.max()) <= 1.0, (what, float(ratio.max()), int(ratio.argmax()))
    empty = count == 0
    assert bool((got[empty] == 0).all()), what


# ------------------------------------------------------------------------------------------------
# rotary
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n,hq,hk,dim,sections,interleaved', [
    (1, 1, 1, 2, [1], False), (1, 8, 8, 16, [3, 3, 2], False), (61, 8, 8, 16, [3, 3, 2], False), (5, 3, 1, 128, [64], False),
    (130, 7, 1, 80, [13, 13, 13], False), (33, 4, 2, 96, [10, 6, 5], False), (700, 2, 1, 64, [16, 8, 8], True),
    (9, 3, 2, 30, [7], True), (9, 3, 2, 30, [7], False), (17, 1, 0, 256, [128], False), (17, 2, 1, 256, [100, 28], True),
    (40, 5, 5, 24, [0, 4, 8], False),
])
def test_rotary(n, hq, hk, dim, sections, interleaved, dtype):
    g = _gen(n + dim)
    x = _rand(g, n, hq + hk + 1, dim, dtype=dtype, scale=2.0)
    qk = x.to(DEV)
    q, k = qk[:, :hq], (qk[:, hq:hq + hk] if hk else None)
    pairs = sum(sections)
    freqs = torch.rand(pairs, generator=g) ** 3
    for pos in (torch.randn(n, len(sections), generator=g) * 300, torch.randint(-5, 1_000_000, (n, len(sections)), generator=g),
                torch.randint(0, 5000, (n, len(sections)), generator=g, dtype=torch.int32)):
        for inverse in (False, True):
            got = ops.rotary_embed(q, k, pos.to(DEV), freqs.to(DEV), sections, interleaved, inverse)
            for part, a, b in ((got[0], 0, hq), (got[1], hq, hq + hk)):
                if a == b:
                    assert part is None
                    continue
                want = ref.rotary(x[:, a:b], pos, freqs, sections, interleaved, inverse)
                tol = ref.rotary_tolerance(dtype, x[:, a:b], want, pairs, interleaved)
                assert part.is_contiguous() and part.dtype == dtype
                assert bool(((part.cpu().double() - want).abs() <= tol).all())
                if not interleaved:
                    assert torch.equal(part[..., 2 * pairs:].cpu(), x[:, a:b, 2 * pairs:])     # passed through, bit for bit
                else:
                    assert torch.equal(part[..., 2 * pairs:].cpu(), x[:, a:b, 2 * pairs:])


def test_rotary_passes_non_finite_features_through_and_keeps_them_in_their_pair():
    x = torch.randn(3, 2, 16, generator=_gen(1))
    x[1, 0, 14], x[1, 1, 3] = float('nan'), float('inf')
    for interleaved in (False, True):
        got, _ = ops.rotary_embed(x.to(DEV), None, torch.arange(3).view(3, 1).to(DEV), torch.ones(5, device=DEV), [5], interleaved)
        want = ref.rotary(x, torch.arange(3).view(3, 1), torch.ones(5), [5], interleaved)
        assert torch.equal(torch.isfinite(got.cpu()), torch.isfinite(want))


def test_rotary_of_strided_and_odd_inputs_and_its_inverse():
    g = _gen(2)
    wide = _rand(g, 50, 4, 41)
    x = wide[:, :, 1:33]                                      # odd row stride, rows 4 bytes off
    pos, freqs = torch.randint(0, 100, (50, 2), generator=g), torch.rand(16, generator=g)
    got, _ = ops.rotary_embed(wide.to(DEV)[:, :, 1:33], None, pos.to(DEV), freqs.to(DEV), [10, 6])
    want = ref.rotary(x, pos, freqs, [10, 6])
    assert bool(((got.cpu().double() - want).abs() <= ref.rotary_tolerance(torch.float32, x, want, 16, False)).all())
    turned = x.transpose(0, 1).contiguous().transpose(0, 1).to(DEV)   # head-major memory
    again, _ = ops.rotary_embed(turned, None, pos.to(DEV), freqs.to(DEV), [10, 6])
    assert torch.equal(again, got)
    back, _ = ops.rotary_embed(got, None, pos.to(DEV), freqs.to(DEV), [10, 6], inverse=True)
    # two rotations: twice the bound of one, on rows whose pairs keep their length (|a| + |b| grows by at most sqrt 2)
    tol = 2 * 1.5 * ref.rotary_tolerance(torch.float32, x, x.double().abs() + 1, 16, False)
    assert bool(((back.cpu().double() - x.double()).abs() <= tol).all())
    empty = ops.rotary_embed(torch.empty(0, 2, 8, device=DEV), torch.empty(0, 1, 8, device=DEV), torch.empty(0, 1, device=DEV),
                             torch.ones(4, device=DEV), [4])
    assert empty[0].shape == (0, 2, 8) and empty[1].shape == (0, 1, 8)


def test_rotary_inverse_is_the_gradient():
    """<g, R x> = <R^T g, x>, against differences in float64 of the definition."""
    g = _gen(3)
    x, up = _rand(g, 6, 2, 16), _rand(g, 6, 2, 16)
    pos, freqs = torch.randn(6, 3, generator=g) * 20, torch.rand(8, generator=g)
    grad, _ = ops.rotary_embed(up.to(DEV), None, pos.to(DEV), freqs.to(DEV), [3, 3, 2], inverse=True)
    h = 1e-3
    for n, hd, i in ((0, 0, 0), (3, 1, 9), (5, 0, 15)):
        e = torch.zeros_like(x, dtype=torch.float64)
        e[n, hd, i] = h
        f = lambda t: float((ref.rotary(t, pos, freqs, [3, 3, 2]) * up.double()).sum())
        slope = (f(x.double() + e) - f(x.double() - e)) / (2 * h)          # linear in x: exact up to float64 rounding
        assert abs(slope - float(grad[n, hd, i])) < 1e-5


# ------------------------------------------------------------------------------------------------
# window attention
# ------------------------------------------------------------------------------------------------
CASES = [
    # lens, extra keys per sequence, hq, hk, dim, window, sinks, masked
    ([1], None, 1, 1, 8, 1, 0, False),
    ([59, 59, 59], None, 8, 8, 16, 10, 1, True),
    ([3, 0, 17, 1, 64, 65], None, 4, 2, 16, 5, 2, False),
    ([33, 1, 100], None, 6, 2, 32, 7, 0, True),
    ([130, 31], None, 7, 1, 64, 50, 3, False),
    ([257], None, 4, 4, 64, 64, 16, True),
    ([200, 5], None, 2, 1, 80, 33, 4, False),
    ([150], None, 3, 3, 96, 1, 0, False),
    ([97, 140], None, 4, 1, 128, 70, 5, True),
    ([300], None, 2, 2, 128, 1000, 4, False),
    ([1, 2, 9], [70, 3, 128], 8, 2, 64, 40, 4, False),
    ([40, 16], [100, 0], 5, 1, 128, 64, 1, True),
    ([20, 30], [-7, -30], 2, 1, 32, 6, 2, False),          # fewer keys than queries: the first rows stand before the first key
    ([70], [200], 2, 1, 48, 1 << 50, 1 << 50, False),
    ([66, 66], None, 1, 1, 24, 2, 65, False),
    # few queries behind long prefixes: the keys are split over blocks and joined
    ([9, 1, 0, 30], [2100, 1500, 64, 0], 2, 1, 64, 1400, 3, False),
    ([1], [3000], 5, 1, 128, 4000, 0, True),
    ([17], [4200], 1, 1, 32, 4100, 70, True),
]


def _case(lens, extra, hq, hk, dim, dtype, masked, seed=0, share=0.8):
    g = _gen(seed + dim + sum(lens))
    lens_k = lens if extra is None else [a + b for a, b in zip(lens, extra)]
    nq, nk = sum(lens), sum(lens_k)
    q, k, v = _rand(g, nq, hq, dim, dtype=dtype, scale=1.5), _rand(g, nk, hk, dim, dtype=dtype), _rand(g, nk, hk, dim, dtype=dtype)
    mask = torch.rand(nk, generator=g) < share if masked else None
    return q, k, v, _cu(lens), (None if extra is None else _cu(lens_k)), mask


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('case', range(len(CASES)))
def test_window(case, dtype):
    lens, extra, hq, hk, dim, win, sinks, masked = CASES[case]
    q, k, v, cu_q, cu_k, mask = _case(lens, extra, hq, hk, dim, dtype, masked)
    dq, dk, dv, dcq, dck, dm = _dev(q, k, v, cu_q, cu_k, mask)
    got = ops.attn_window(dq, dk, dv, dcq, win, sinks, cu_k=dck, key_mask=dm)
    _check(got, ref.window(q, k, v, cu_q, win, sinks, cu_k, mask), dtype, dim, v)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [16, 64, 128])
def test_window_views_scale_and_rows_behind_the_last_sequence(dim, dtype):
    g = _gen(dim)
    lens, hq, hk = [37, 90], 4, 2
    n, behind = sum(lens), 11
    qkv = _rand(g, n + behind, hq + 2 * hk, dim, dtype=dtype)
    cu = _cu(lens)
    d = qkv.to(DEV)
    got = ops.attn_window(d[:, :hq], d[:, hq:hq + hk], d[:, hq + hk:], cu.to(DEV), 20, 2, scale=0.37)
    q, k, v = qkv[:n, :hq], qkv[:n, hq:hq + hk], qkv[:n, hq + hk:]
    _check(got[:n], ref.window(q, k, v, cu, 20, 2, scale=0.37), dtype, dim, v)
    assert bool((got[n:] == 0).all())
    odd = _rand(g, n, hq, dim + 1, dtype=dtype)                          # rows that are not 16-byte aligned: copied
    dk, dv = k.contiguous().to(DEV), v.contiguous().to(DEV)
    a = ops.attn_window(odd.to(DEV)[..., :dim], dk, dv, cu.to(DEV), 20, 2)
    _check(a, ref.window(odd[..., :dim], k, v, cu, 20, 2), dtype, dim, v)
    flat = ops.attn_window(odd.to(DEV)[..., :dim], dk, dv, cu.to(DEV), 20, 2, scale=0.0)      # scale 0: the plain mean
    _check(flat, ref.window(odd[..., :dim], k, v, cu, 20, 2, scale=0.0), dtype, dim, v)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim,hq,hk', [(16, 8, 8), (64, 4, 2), (128, 4, 1)])
def test_window_ignores_what_masked_and_unseen_places_hold(dim, hq, hk, dtype):
    """NaN and infinities in keys and values that a row does not see change nothing for it: masked ones for all rows, later and
    older ones for the rows that do not reach them."""
    lens = [150, 70]
    q, k, v, cu, _, mask = _case(lens, None, hq, hk, dim, dtype, True, seed=5)
    want = ref.window(q, k, v, cu, 40, 2, None, mask)
    for fill in (float('nan'), float('inf'), -float('inf')):
        kk, vv = k.clone(), v.clone()
        kk[~mask], vv[~mask] = fill, fill
        _check(ops.attn_window(*_dev(q, kk, vv, cu), 40, 2, key_mask=mask.to(DEV)), want, dtype, dim, v, fill)
        # one visible key's value is not finite: only the rows that see it (positions 30 .. 69 of the first sequence) follow
        mask2 = mask.clone()
        mask2[30] = True
        vv[30] = fill
        got = ops.attn_window(*_dev(q, kk if mask[30] else torch.where(torch.arange(220)[:, None, None] == 30, k, kk), vv, cu), 40, 2,
                              key_mask=mask2.to(DEV)).cpu()
        sees = torch.zeros(220, dtype=torch.bool)
        sees[30:70] = True
        assert not bool(torch.isfinite(got[sees]).any())
        w2 = ref.window(q, k, v, cu, 40, 2, None, mask)
        if bool(mask[30]):
            keep = ~sees
            tol = ref.tolerance(dtype, dim, *w2, float(v.double().abs().max()))
            assert bool(((got.double() - w2[0]).abs() <= tol)[keep].all())
        else:
            assert bool(torch.isfinite(got[~sees]).all())


@pytest.mark.parametrize('dtype', DTYPES)
def test_window_split_over_blocks_with_rows_behind_and_unseen_infinities(dtype):
    lens, extra, hq, hk, dim = [20, 6], [2500, 1100], 2, 1, 64
    q, k, v, cu_q, cu_k, mask = _case(lens, extra, hq, hk, dim, dtype, True, seed=8)
    behind = 5
    qq = torch.cat([q, torch.ones(behind, hq, dim, dtype=dtype)])
    want = ref.window(q, k, v, cu_q, 2200, 2, cu_k, mask)
    vv = v.clone()
    vv[~mask] = float('nan')
    last = int(cu_k[1]) - 3                                    # seen by the first sequence's last three queries only
    mask2 = mask.clone()
    mask2[last] = True
    vv[last] = float('inf')
    got = ops.attn_window(*_dev(qq, k, vv, cu_q), 2200, 2, cu_k=cu_k.to(DEV), key_mask=mask2.to(DEV)).cpu().double()
    assert bool((got[26:] == 0).all())
    keep = torch.ones(26, dtype=torch.bool)
    keep[17:20] = False
    assert not bool(torch.isfinite(got[17:20]).any())
    tol = ref.tolerance(dtype, dim, *want, float(v.double().abs().max()))
    assert bool(((got[:26] - want[0]).abs() <= tol)[keep].all())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lens,extra,hq,hk,dim,win', [([40, 23], None, 4, 2, 16, 50), ([150, 70], None, 4, 2, 64, 120),
                                                      ([20, 6], [2500, 1100], 2, 1, 64, 2200)])
def test_window_nan_reaches_the_rows_that_see_it(lens, extra, hq, hk, dim, win, dtype):
    """A NaN in a query makes that row NaN and no other; a stretch of NaN keys, longer than what one block of a split works on, every
    row that sees it."""
    q, k, v, cu_q, cu_k, _ = _case(lens, extra, hq, hk, dim, dtype, False, seed=13)
    cuk = None if extra is None else cu_k.to(DEV)
    want = ref.window(q, k, v, cu_q, win, 1, cu_k)
    tol = ref.tolerance(dtype, dim, *want, float(v.double().abs().max()))
    qq = q.clone()
    qq[3, 1, 5] = float('nan')
    got = ops.attn_window(*_dev(qq, k, v, cu_q), win, 1, cu_k=cuk).cpu().double()
    assert bool(got[3, 1].isnan().all())
    got[3, 1] = want[0][3, 1]
    assert bool(((got - want[0]).abs() <= tol).all())
    kk = k.clone()
    kk[: lens[0] - 5 if extra is None else 1300] = float('nan')    # the sink and more, of the first sequence: all its rows see some
    got = ops.attn_window(*_dev(q, kk, v, cu_q), win, 1, cu_k=cuk).cpu().double()
    n0 = lens[0]
    assert bool(got[:n0].isnan().all())
    assert bool(((got - want[0]).abs() <= tol)[n0:].all())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [16, 64])
def test_window_rows_more_than_4_gib_apart(dim, dtype):
    """Token strides just below the limit: offsets of 80 tokens pass 32 bits, in bytes for float32 and in signed elements for all."""
    n, h, tok = 80, 2, (1 << 24) - 16
    q, k, v, cu, _, mask = _case([50, 30], None, h, h, dim, dtype, True, seed=14)
    room = torch.empty(n * tok, dtype=dtype, device=DEV)
    views = [room.as_strided((n, h, dim), (tok, 4096, 1), 65536 * i) for i in range(3)]      # interleaved in one stretch of memory
    for view, x in zip(views, (q, k, v)):
        view.copy_(x)
    got = ops.attn_window(*views, cu.to(DEV), 20, 2, key_mask=mask.to(DEV))
    _check(got, ref.window(q, k, v, cu, 20, 2, key_mask=mask), dtype, dim, v)
    tq, tk = ops.rotary_embed(views[0], views[1], torch.arange(n, device=DEV).view(n, 1), torch.ones(dim // 2, device=DEV), [dim // 2])
    sq, sk = ops.rotary_embed(q.to(DEV), k.to(DEV), torch.arange(n, device=DEV).view(n, 1), torch.ones(dim // 2, device=DEV), [dim // 2])
    assert torch.equal(tq, sq) and torch.equal(tk, sk)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('win', [1100, 1700, 4000])
@pytest.mark.parametrize('dim', [24, 40, 128])
def test_window_split_into_few_and_many_parts_of_an_odd_number_of_rows(dim, win, dtype):
    """81 rows in two, three and seven parts of the keys (the join takes one or two rows per wave); an infinity that two rows of three
    heads see makes them, and only them, infinite or NaN."""
    lens, extra, hq = [21, 6], [4000, 900], 3
    q, k, v, cu_q, cu_k, mask = _case(lens, extra, hq, hq, dim, dtype, True, seed=50)
    want = ref.window(q, k, v, cu_q, win, 2, cu_k, mask)
    tol = ref.tolerance(dtype, dim, *want, float(v.double().abs().max()))
    args = _dev(q, k, v, cu_q)
    got = ops.attn_window(*args, win, 2, cu_k=cu_k.to(DEV), key_mask=mask.to(DEV)).cpu().double()
    assert bool(((got - want[0]).abs() <= tol).all())
    vv, seen = v.clone(), mask.clone()
    vv[int(cu_k[1]) - 2] = float('inf')                        # the first sequence's last two queries reach it
    seen[int(cu_k[1]) - 2] = True
    got = ops.attn_window(args[0], args[1], vv.to(DEV), args[3], win, 2, cu_k=cu_k.to(DEV), key_mask=seen.to(DEV)).cpu().double()
    assert not bool(torch.isfinite(got[19:21]).any())
    keep = torch.ones(27, dtype=torch.bool)
    keep[19:21] = False
    assert bool(((got - want[0]).abs() <= tol)[keep].all())


@pytest.mark.parametrize('dtype', DTYPES)
def test_window_all_masked_and_large_scores(dtype):
    q, k, v, cu, _, _ = _case([45, 30], None, 4, 2, 32, dtype, False, seed=6)
    none = torch.zeros(75, dtype=torch.bool)
    assert bool((ops.attn_window(*_dev(q, k, v, cu), 9, 1, key_mask=none.to(DEV)) == 0).all())
    # scores of several thousands: the running maximum moves by far more than any exponent range
    q2, k2 = q * 40, k * 40
    q2, k2 = q2.to(dtype), k2.to(dtype)
    r = ref.window(q2, k2, v, cu, 30, 1)
    got = ops.attn_window(*_dev(q2, k2, v, cu), 30, 1).cpu().double()
    assert bool(torch.isfinite(got).all())
    tol = ref.tolerance(dtype, 32, *r, float(v.double().abs().max()))
    assert bool(((got - r[0]).abs() <= tol).all())


def test_window_bad_boundaries_stay_inside():
    """Boundaries that are wrong on the device give wrong rows, not wild accesses; the right sequences of a next call are right."""
    q, k, v, cu, _, _ = _case([45, 30], None, 4, 2, 64, torch.bfloat16, False, seed=7)
    dq, dk, dv = _dev(q, k, v)
    for bad in ([0, 100, 50], [0, 40, 1 << 40], [0, -5, 75], [75, 0, 75]):
        out = ops.attn_window(dq, dk, dv, torch.tensor(bad, device=DEV), 9, 1)
        assert out.shape == q.shape
    torch.cuda.synchronize()
    _check(ops.attn_window(dq, dk, dv, cu.to(DEV), 9, 1), ref.window(q, k, v, cu, 9, 1), torch.bfloat16, 64, v)


def test_window_of_nothing():
    e = lambda *s: torch.empty(*s, device=DEV)
    z = torch.zeros(1, dtype=torch.int64, device=DEV)
    assert ops.attn_window(e(0, 2, 16), e(0, 2, 16), e(0, 2, 16), z, 4).shape == (0, 2, 16)
    # queries without any key are rows that see nothing; no sequence at all: rows behind the last one
    got = ops.attn_window(torch.ones(5, 2, 16, device=DEV), e(0, 2, 16), e(0, 2, 16), torch.tensor([0, 5], device=DEV), 4,
                          cu_k=torch.tensor([0, 0], device=DEV))
    assert bool((got == 0).all())
    assert bool((ops.attn_window(*[torch.ones(5, 2, 16, device=DEV)] * 3, z, 4) == 0).all())


# ------------------------------------------------------------------------------------------------
# cache
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lens,ages,hk,dim,win,sinks,masked', [
    ([1], [0], 1, 8, 1, 0, False), ([5, 0, 40, 1], [0, 7, 3, 100], 2, 16, 6, 2, True), ([59] * 5, [0] * 5, 8, 16, 50, 1, True),
    ([100, 33, 17], [0, 1 << 40, 15], 3, 128, 20, 4, False), ([70, 9], [2, -1], 2, 80, 64, 3, True),
    ([16, 16, 32], [1, 2, 3], 1, 64, 3, 16, False),
])
def test_append(lens, ages, hk, dim, win, sinks, masked, dtype):
    g = _gen(sum(lens))
    n, b, slots = sum(lens), len(lens), win + sinks
    behind = 3
    k, v = _rand(g, n + behind, hk, dim, dtype=dtype), _rand(g, n + behind, hk, dim, dtype=dtype)
    kc, vc = _rand(g, b, hk, slots, dim, dtype=dtype), _rand(g, b, hk, slots, dim, dtype=dtype)
    mc = torch.rand(b, slots, generator=g) < 0.5 if masked else None
    km = torch.rand(n + behind, generator=g) < 0.5 if masked else None
    cu, lengths = _cu(lens), torch.tensor(ages)
    dk, dv, dcu, dl, dkc, dvc, dkm, dmc = _dev(k, v, cu, lengths, kc, vc, km, mc)
    ops.window_cache_append(dk, dv, dcu, dl, dkc, dvc, sinks, key_mask=dkm, mask_cache=dmc)
    ref.append(k, v, cu, lengths, kc, vc, sinks, km, mc)
    assert torch.equal(dkc.cpu(), kc) and torch.equal(dvc.cpu(), vc) and torch.equal(dl.cpu(), lengths)
    assert mc is None or torch.equal(dmc.cpu(), mc)


STEPS = [
    # batch ages, hq, hk, dim, window, sinks, masked
    ([0], 1, 1, 8, 1, 0, False),
    ([0, 1, 5, 49, 50, 51, 300, -1], 8, 8, 16, 50, 1, True),
    ([3, 700, 0], 4, 2, 32, 100, 4, False),
    ([20000, 15, 257], 7, 1, 64, 260, 3, True),
    ([1000, 1 << 41], 16, 1, 80, 65, 0, False),
    ([129, 64, 5000], 20, 1, 96, 130, 16, True),
    ([4103, 0, 4200, -7, 2000], 8, 2, 128, 1500, 4, False),
    ([6000], 4, 1, 128, 4096, 4, False),
    ([9000, 8000], 40, 2, 64, 2500, 0, True),
]


def _step_case(ages, hq, hk, dim, win, sinks, masked, dtype, seed=0):
    g = _gen(seed + dim + win)
    b, slots = len(ages), win + sinks
    q, k, v = _rand(g, b, hq, dim, dtype=dtype, scale=1.5), _rand(g, b, hk, dim, dtype=dtype), _rand(g, b, hk, dim, dtype=dtype)
    kc, vc = _rand(g, b, hk, slots, dim, dtype=dtype), _rand(g, b, hk, slots, dim, dtype=dtype)
    mc = torch.rand(b, slots, generator=g) < 0.8 if masked else None
    km = torch.rand(b, generator=g) < 0.6 if masked else None
    return q, k, v, torch.tensor(ages), kc, vc, km, mc


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('case', range(len(STEPS)))
def test_step(case, dtype):
    ages, hq, hk, dim, win, sinks, masked = STEPS[case]
    q, k, v, lengths, kc, vc, km, mc = _step_case(ages, hq, hk, dim, win, sinks, masked, dtype)
    # slots that no position has filled hold what they hold
    for b, age in enumerate(ages):
        if 0 <= age < win + sinks - 1:
            kc[b, :, age + 1:], vc[b, :, age + 1:] = float('nan'), float('nan')
    dq, dk, dv, dl, dkc, dvc, dkm, dmc = _dev(q, k, v, lengths, kc, vc, km, mc)
    got = ops.attn_window_step(dq, dk, dv, dl, dkc, dvc, sinks, key_mask=dkm, mask_cache=dmc)
    r = ref.step(q, k, v, lengths, kc, vc, sinks, km, mc)
    _check(got, r, dtype, dim, torch.cat([torch.nan_to_num(vc.double()).abs().amax().view(1)]))
    same = lambda a, b: torch.equal(torch.nan_to_num(a.cpu(), 7.0), torch.nan_to_num(b, 7.0))
    assert same(dkc, kc) and same(dvc, vc) and torch.equal(dl.cpu(), lengths)
    assert mc is None or torch.equal(dmc.cpu(), mc)


@pytest.mark.parametrize('dtype', DTYPES)
def test_step_ignores_what_masked_slots_hold(dtype):
    q, k, v, lengths, kc, vc, km, mc = _step_case([500, 40, 7], 8, 2, 64, 300, 4, True, dtype, seed=3)
    for fill in (float('nan'), float('inf')):
        a, b = kc.clone(), vc.clone()
        a.masked_fill_(~mc[:, None, :, None], fill)
        b.masked_fill_(~mc[:, None, :, None], fill)
        dkc, dvc, dmc = _dev(a, b, mc)
        got = ops.attn_window_step(*_dev(q, k, v, lengths), dkc, dvc, 4, key_mask=km.to(DEV), mask_cache=dmc)
        _check(got, ref.step(q, k, v, lengths, kc.clone(), vc.clone(), 4, km, mc.clone()), dtype, 64, vc, fill)
    gone = torch.zeros_like(mc).to(DEV)
    got = ops.attn_window_step(*_dev(q, k, v, lengths, kc, vc), 4, key_mask=torch.zeros(3, dtype=torch.bool, device=DEV), mask_cache=gone)
    assert bool((got == 0).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16])
def test_cache_rows_beyond_4_gib(dtype):
    """The second row of a cache whose rows are more than 4 GiB each: prompt and step land there and read there, and a length that
    has gone round the ring comes back to its start."""
    hk, dim, sinks = 1, 128, 2
    slots = (1 << 32) // (dim * torch.finfo(dtype).bits // 8) + 70
    kc, vc = (torch.empty(2, hk, slots, dim, dtype=dtype, device=DEV) for _ in range(2))
    g = _gen(15)
    n = 40
    k, v = _rand(g, n, hk, dim, dtype=dtype), _rand(g, n, hk, dim, dtype=dtype)
    q, k1, v1 = _rand(g, 2, 2, dim, dtype=dtype), _rand(g, 2, hk, dim, dtype=dtype), _rand(g, 2, hk, dim, dtype=dtype)
    lengths = torch.tensor([-1, 0])
    ops.window_cache_append(*_dev(k, v), torch.tensor([0, 0, n], device=DEV), lengths.to(DEV), kc, vc, sinks)
    assert torch.equal(kc[1, 0, :n].cpu(), k[:, 0]) and torch.equal(vc[1, 0, :n].cpu(), v[:, 0])
    lengths[1] = n
    got = ops.attn_window_step(*_dev(q, k1, v1, lengths), kc, vc, sinks)
    assert torch.equal(kc[1, 0, n].cpu(), k1[1, 0]) and torch.equal(vc[1, 0, n].cpu(), v1[1, 0])
    allk, allv = torch.cat([k, k1[1:]]), torch.cat([v, v1[1:]])
    want = ref.window(torch.cat([torch.zeros(n, 2, dim, dtype=dtype), q[1:]]), allk, allv, torch.tensor([0, n + 1]), slots, sinks)
    assert bool((got[0] == 0).all())
    _check(got[1:], [x[n:] for x in want], dtype, dim, allv)
    ops.window_cache_append(*_dev(k, v), torch.tensor([0, 0, n], device=DEV), torch.tensor([-1, slots - 7], device=DEV), kc, vc, sinks)
    assert torch.equal(kc[1, 0, slots - 7:].cpu(), k[:7, 0]) and torch.equal(vc[1, 0, sinks:sinks + n - 7].cpu(), v[7:, 0])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('win', [20, 700])
def test_step_nan_query(win, dtype):
    q, k, v, lengths, kc, vc, _, _ = _step_case([900, 90], 4, 2, 64, win, 3, False, dtype, seed=16)
    want = ref.step(q, k, v, lengths, kc.clone(), vc.clone(), 3)
    qq = q.clone()
    qq[0, 2, 9] = float('nan')
    got = ops.attn_window_step(*_dev(qq, k, v, lengths, kc, vc), 3).cpu().double()
    assert bool(got[0, 2].isnan().all())
    got[0, 2] = want[0][0, 2]
    assert bool(((got - want[0]).abs() <= ref.tolerance(dtype, 64, *want, float(vc.double().abs().max()))).all())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim,hq,hk,win,sinks', [(8, 5, 5, 10, 1), (24, 6, 2, 16, 1), (32, 8, 8, 10, 1), (32, 3, 3, 17, 0), (32, 12, 4, 1, 16),
                                                 (32, 7, 1, 18, 0), (24, 4, 4, 1, 0)])
def test_window_narrow_heads_and_short_windows(dim, hq, hk, win, sinks, dtype):
    """Windows on both sides of what one step of 32 keys holds, heads that do not fill a 128-byte line, masked keys that hold NaN."""
    q, k, v, cu, _, mask = _case([59, 1, 0, 16, 130, 17], None, hq, hk, dim, dtype, True, seed=30)
    kk, vv = k.clone(), v.clone()
    kk[~mask], vv[~mask] = float('nan'), float('inf')
    got = ops.attn_window(*_dev(q, kk, vv, cu), win, sinks, key_mask=mask.to(DEV))
    _check(got, ref.window(q, k, v, cu, win, sinks, None, mask), dtype, dim, v)
    _check(ops.attn_window(*_dev(q, k, v, cu), win, sinks), ref.window(q, k, v, cu, win, sinks), dtype, dim, v)
    vv = v.clone()
    vv[70] = float('inf')                                      # seen by some rows of a tile only
    got = ops.attn_window(*_dev(q, k, vv, cu), win, sinks).cpu().double()
    r = ref.window(q, k, v, cu, win, sinks)
    tol = ref.tolerance(dtype, dim, *r, float(v.double().abs().max()))
    at = torch.arange(223)
    sees = (at >= 70) & (at < 76) & (at < 70 + win) if 70 - 60 >= sinks else (at >= 70) & (at < 76)
    assert not bool(torch.isfinite(got[sees]).any())
    assert bool(((got - r[0]).abs() <= tol)[~sees].all())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('slots', [240, 256, 257])
@pytest.mark.parametrize('batch,hq,hk,dim', [(3, 8, 2, 64), (70, 8, 8, 16)])
def test_step_around_the_size_that_one_wave_takes(batch, hq, hk, dim, slots, dtype):
    ages = [(37 * i) % (2 * slots) for i in range(batch)]
    q, k, v, lengths, kc, vc, km, mc = _step_case(ages, hq, hk, dim, slots - 2, 2, True, dtype, seed=31)
    dkc, dvc, dmc = _dev(kc, vc, mc)
    got = ops.attn_window_step(*_dev(q, k, v, lengths), dkc, dvc, 2, key_mask=km.to(DEV), mask_cache=dmc)
    _check(got, ref.step(q, k, v, lengths, kc, vc, 2, km, mc), dtype, dim, vc)
    assert torch.equal(dkc.cpu(), kc) and torch.equal(dvc.cpu(), vc) and torch.equal(dmc.cpu(), mc)


def test_lengths_out_of_range_are_rows_not_in_use():
    q, k, v, _, kc, vc, _, _ = _step_case([5, 5], 4, 2, 64, 20, 3, False, torch.bfloat16, seed=17)
    lengths = torch.tensor([(1 << 63) - 1, (1 << 62) + 1], device=DEV)
    dq, dk, dv, dkc, dvc = _dev(q, k, v, kc, vc)
    assert bool((ops.attn_window_step(dq, dk, dv, lengths, dkc, dvc, 3) == 0).all())
    ops.window_cache_append(dk, dv, torch.tensor([0, 1, 2], device=DEV), lengths, dkc, dvc, 3)
    assert torch.equal(dkc.cpu(), kc) and torch.equal(dvc.cpu(), vc)


def test_caches_that_share_memory_are_refused():
    room = torch.zeros(3, 1, 8, 16, device=DEV)
    x, n = torch.zeros(2, 1, 16, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    for a, b in ((room[:2], room[:2]), (room[:2], room[1:])):
        with pytest.raises(ValueError, match='share memory'):
            ops.attn_window_step(x, x, x, n, a, b, 1)
        with pytest.raises(ValueError, match='share memory'):
            ops.window_cache_append(x, x, torch.tensor([0, 1, 2], device=DEV), n, a, b, 1)


# ------------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('hq,hk,dim,win,sinks', [(8, 8, 16, 10, 1), (8, 2, 64, 24, 4)])
def test_prefill_append_and_steps_are_the_whole_sequence(hq, hk, dim, win, sinks, dtype):
    """Rotate, attend and cache a ragged prefix, then rotate + step token by token (one row leaves the batch on the way): every
    step's output is the row that one pass over the whole sequence gives."""
    g = _gen(11)
    prefix, more = [31, 5, 0], 9
    lens = [p + more for p in prefix]
    n = sum(lens)
    qkv = _rand(g, n, hq + 2 * hk, dim, dtype=dtype).to(DEV)
    mask = (torch.rand(n, generator=g) < 0.8).to(DEV)
    cu = _cu(lens).to(DEV)
    pos = torch.cat([torch.arange(m) for m in lens]).view(n, 1).to(DEV)
    freqs = torch.rand(dim // 2, generator=g).to(DEV)
    q, k = ops.rotary_embed(qkv[:, :hq], qkv[:, hq:hq + hk], pos, freqs, [dim // 2])
    v = qkv[:, hq + hk:]
    want = ref.window(q.cpu(), k.cpu(), v.cpu(), cu.cpu(), win, sinks, key_mask=mask.cpu())
    _check(ops.attn_window(q, k, v, cu, win, sinks, key_mask=mask), want, dtype, dim, v)
    starts = cu[:-1].tolist()
    rows = torch.cat([torch.arange(s, s + m) for s, m in zip(starts, prefix)]).to(DEV)
    b = len(lens)
    kc, vc = torch.zeros(b, hk, win + sinks, dim, dtype=dtype, device=DEV), torch.zeros(b, hk, win + sinks, dim, dtype=dtype, device=DEV)
    mc = torch.zeros(b, win + sinks, dtype=torch.bool, device=DEV)
    lengths = torch.zeros(b, dtype=torch.int64, device=DEV)
    ops.window_cache_append(k[rows], v[rows], _cu(prefix).to(DEV), lengths, kc, vc, sinks, key_mask=mask[rows], mask_cache=mc)
    lengths += torch.tensor(prefix, device=DEV)
    tol = ref.tolerance(dtype, dim, *want, float(v.double().abs().max()))
    for t in range(more):
        at = torch.tensor([s + p + t for s, p in zip(starts, prefix)], device=DEV)
        used = lengths.clone()
        if t >= 5:
            used[1] = -1
        qt, kt = ops.rotary_embed(qkv[at, :hq], qkv[at, hq:hq + hk], pos[at], freqs, [dim // 2])
        got = ops.attn_window_step(qt, kt, v[at], used, kc, vc, sinks, key_mask=mask[at], mask_cache=mc).cpu().double()
        for r in range(b):
            if r == 1 and t >= 5:
                assert bool((got[r] == 0).all())
            else:
                assert bool(((got[r] - want[0][at[r]]).abs() <= tol[at[r]]).all()), (t, r)
        lengths += 1


def test_steps_in_a_graph_on_another_stream():
    """A captured decoding step (rotate, step, advance the lengths), replayed with eager work in between, equals the eager run."""
    g = _gen(12)
    b, hq, hk, dim, win, sinks = 3, 8, 2, 128, 600, 4
    dtype = torch.bfloat16
    freqs = torch.rand(64, generator=g).to(DEV)
    kc0, vc0 = _rand(g, b, hk, win + sinks, dim, dtype=dtype).to(DEV), _rand(g, b, hk, win + sinks, dim, dtype=dtype).to(DEV)
    tokens = _rand(g, 5, b, hq + 2 * hk, dim, dtype=dtype).to(DEV)
    start = torch.tensor([0, 590, 3000], device=DEV)

    def one(x, lengths, kc, vc):
        q, k = ops.rotary_embed(x[:, :hq], x[:, hq:hq + hk], lengths.view(b, 1), freqs, [64])
        out = ops.attn_window_step(q, k, x[:, hq + hk:], lengths, kc, vc, sinks)
        lengths += 1
        return out

    kc, vc, lengths = kc0.clone(), vc0.clone(), start.clone()
    eager = [one(tokens[i], lengths, kc, vc).clone() for i in range(5)]
    gk, gv, gl, x = kc0.clone(), vc0.clone(), start.clone(), tokens[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(x, gl, gk, gv)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one(x, gl, gk, gv)
    gk.copy_(kc0), gv.copy_(vc0), gl.copy_(start)
    for i in range(5):
        x.copy_(tokens[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i]), i
        ops.attn_window_step(tokens[0, :, :hq], tokens[0, :, hq:hq + hk], tokens[0, :, hq + hk:], start, kc0.clone(), vc0.clone(), sinks)
    assert torch.equal(gk, kc) and torch.equal(gv, vc) and torch.equal(gl, lengths)


@pytest.mark.parametrize('lens,extra,win', [([300, 45], None, 60), ([20, 6], [2500, 1100], 2200)])
def test_prefill_in_a_graph(lens, extra, win):
    """Rotation, attention (in one pass and split over blocks) and append, captured once and replayed on other data, with eager calls in
    between, equal the eager calls."""
    hq, hk, dim, sinks, dtype = 4, 2, 64, 2, torch.bfloat16
    cases = [_case(lens, extra, hq, hk, dim, dtype, True, seed=20 + i) for i in range(3)]
    cu_q, cu_k = _dev(cases[0][3], cases[0][4] if extra is not None else cases[0][3])
    nq, nk = cases[0][0].size(0), cases[0][1].size(0)
    freqs, pos = torch.rand(dim // 2, generator=_gen(21)).to(DEV), torch.arange(nq, device=DEV).view(nq, 1)
    lengths = torch.tensor([3, 0], device=DEV)

    def one(q, k, v, mask, kc, vc, mc):
        q = ops.rotary_embed(q, None, pos, freqs, [dim // 2])[0]
        out = ops.attn_window(q, k, v, cu_q, win, sinks, cu_k=cu_k, key_mask=mask)
        ops.window_cache_append(k, v, cu_k, lengths, kc, vc, sinks, key_mask=mask, mask_cache=mc)
        return out

    def cache():
        return (torch.zeros(2, hk, win + sinks, dim, dtype=dtype, device=DEV), torch.zeros(2, hk, win + sinks, dim, dtype=dtype, device=DEV),
                torch.zeros(2, win + sinks, dtype=torch.bool, device=DEV))

    data = [_dev(c[0], c[1], c[2], c[5]) for c in cases]
    wants = []
    for d in data:
        c = cache()
        wants.append((one(*d, *c).clone(), c))
    held, kept = [x.clone() for x in data[0]], cache()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(*held, *kept)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one(*held, *kept)
    for _ in range(2):
        for d, (want, c) in zip(data, wants):
            for a, b in zip(held, d):
                a.copy_(b)
            for x in kept:
                x.zero_()
            graph.replay()
            one(*data[0], *cache())
            torch.cuda.synchronize()
            assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(kept, c))


def test_window_on_two_streams_is_the_same_every_time():
    q, k, v, cu, _, mask = _case([300, 45, 170], None, 8, 2, 64, torch.bfloat16, True, seed=9)
    dq, dk, dv, dcu, dm = _dev(q, k, v, cu, mask)
    first = ops.attn_window(dq, dk, dv, dcu, 60, 2, key_mask=dm)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs += [ops.attn_window(dq, dk, dv, dcu, 60, 2, key_mask=dm) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


# ------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------
def test_refusals():
    f = lambda *s, **kw: torch.zeros(*s, device=DEV, **kw)
    i = lambda *s: torch.zeros(*s, dtype=torch.int64, device=DEV)
    cu = torch.tensor([0, 4], device=DEV)
    q, kv = f(4, 4, 16), f(4, 2, 16)
    with pytest.raises(ValueError):
        ops.attn_window(q, kv, f(4, 2, 24), cu, 4)
    with pytest.raises(ValueError):
        ops.attn_window(f(4, 3, 16), kv, kv, cu, 4)
    with pytest.raises(ValueError):
        ops.attn_window(q, kv, kv, cu, 0)
    with pytest.raises(ValueError):
        ops.attn_window(q, kv, kv, cu, 4, -1)
    with pytest.raises(ValueError):
        ops.attn_window(q, f(5, 2, 16), f(5, 2, 16), cu, 4)
    with pytest.raises(TypeError):
        ops.attn_window(q, kv, kv, cu.int(), 4)
    with pytest.raises(TypeError):
        ops.attn_window(q, kv.half(), kv.half(), cu, 4)
    with pytest.raises(TypeError):
        ops.attn_window(q.double(), kv.double(), kv.double(), cu, 4)
    with pytest.raises(_lib.QcnError):
        ops.attn_window(f(4, 4, 20), f(4, 2, 20), f(4, 2, 20), cu, 4)
    with pytest.raises(_lib.QcnError):
        ops.attn_window(f(4, 4, 136), f(4, 2, 136), f(4, 2, 136), cu, 4)
    for bad in (float('nan'), float('inf'), -1.0):
        with pytest.raises(ValueError):
            ops.attn_window(q, kv, kv, cu, 4, scale=bad)
    with pytest.raises(ValueError):
        ops.attn_window(q, kv, kv, cu, 4, key_mask=f(3, dtype=torch.bool))
    with pytest.raises(_lib.QcnError):
        ops.attn_window(q.cpu(), kv.cpu(), kv.cpu(), cu.cpu(), 4)
    cache = lambda: f(4, 2, 6, 16)
    one = cache()
    with pytest.raises(ValueError):
        ops.attn_window_step(q, kv, kv, i(4), cache(), cache(), 6)                       # no slot left for the window
    with pytest.raises(ValueError):
        ops.attn_window_step(q, kv, kv, i(3), cache(), cache(), 1)
    with pytest.raises(ValueError):
        ops.attn_window_step(q, kv, kv, i(4), one, one, 1)
    with pytest.raises(ValueError):
        ops.attn_window_step(q, kv, kv, i(4), f(4, 2, 16, 6).transpose(2, 3), cache(), 1)    # not contiguous
    with pytest.raises(ValueError):
        ops.attn_window_step(q, kv, kv, i(4), cache(), cache(), 1, key_mask=f(4, dtype=torch.bool))
    with pytest.raises(ValueError):
        ops.attn_window_step(q, kv, kv, i(4), cache(), cache(), 1, mask_cache=f(6, 4, dtype=torch.bool).t())
    with pytest.raises(TypeError):
        ops.attn_window_step(q, kv, kv, i(4).int(), cache(), cache(), 1)
    with pytest.raises(ValueError):
        ops.window_cache_append(kv, kv, cu, i(2), f(1, 2, 6, 16), f(1, 2, 6, 16), 1)
    with pytest.raises(TypeError):
        ops.window_cache_append(kv, kv, cu, i(1), f(1, 2, 6, 16).half(), f(1, 2, 6, 16).half(), 1)
    pos = i(4, 2)
    with pytest.raises(ValueError):
        ops.rotary_embed(q, None, pos, f(9), [5, 4])
    with pytest.raises(ValueError):
        ops.rotary_embed(q, None, pos, f(8), [8])
    with pytest.raises(TypeError):
        ops.rotary_embed(q, None, pos.double(), f(8), [4, 4])
    with pytest.raises(ValueError):
        ops.rotary_embed(q, f(4, 2, 24), pos, f(8), [4, 4])
    with pytest.raises(_lib.QcnError):
        ops.rotary_embed(f(4, 2, 15), None, pos, f(4), [2, 2])
    with pytest.raises(ValueError):
        ops.rotary_embed(q, None, pos, f(0), [0, 0])


def test_a_traced_step_is_one_graph():
    """torch.compile (no code generation: backend aot_eager) takes rotation, prefill, append and step in one graph, with the caches
    written in place, and gives what the eager calls give."""
    hq, hk, dim, win, sinks, dtype = 4, 2, 64, 24, 2, torch.bfloat16
    q, k, v, cu, _, mask = _case([30, 17], None, hq, hk, dim, dtype, True, seed=40)
    dq, dk, dv, dcu, dm = _dev(q, k, v, cu, mask)
    pos, freqs = torch.arange(47, device=DEV).view(47, 1), torch.rand(dim // 2, generator=_gen(41)).to(DEV)
    lengths = torch.tensor([30, 17], device=DEV)

    def run(q, k, v, kc, vc, mc):
        q, k = ops.rotary_embed(q, k, pos, freqs, [dim // 2])
        out = ops.attn_window(q, k, v, dcu, win, sinks, key_mask=dm)
        ops.window_cache_append(k, v, dcu, torch.zeros_like(lengths), kc, vc, sinks, key_mask=dm, mask_cache=mc)
        return out, ops.attn_window_step(q[:2], k[:2], v[:2], lengths, kc, vc, sinks, key_mask=dm[:2], mask_cache=mc)

    def cache():
        return (torch.zeros(2, hk, win + sinks, dim, dtype=dtype, device=DEV), torch.zeros(2, hk, win + sinks, dim, dtype=dtype, device=DEV),
                torch.zeros(2, win + sinks, dtype=torch.bool, device=DEV))

    a, b = cache(), cache()
    want = run(dq, dk, dv, *a)
    got = torch.compile(run, backend='aot_eager', fullgraph=True)(dq, dk, dv, *b)
    assert all(torch.equal(x, y) for x, y in zip(got + b, want + a))


def test_sequence_ops_trace_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(40, 12, 64, device=DEV, dtype=torch.bfloat16)
        q, k = ops.rotary_embed(x[:, :8], x[:, 8:10], torch.empty(40, 1, device=DEV), torch.empty(32, device=DEV), [32])
        assert q.shape == (40, 8, 64) and k.shape == (40, 2, 64) and q.dtype == torch.bfloat16
        o = ops.attn_window(q, k, x[:, 10:], torch.empty(3, dtype=torch.int64, device=DEV), 8, 1)
        assert o.shape == (40, 8, 64) and o.dtype == torch.bfloat16
        c = torch.empty(40, 2, 9, 64, device=DEV, dtype=torch.bfloat16)
        assert ops.attn_window_step(q, k, k, torch.empty(40, dtype=torch.int64, device=DEV), c, c.clone(), 1).shape == (40, 8, 64)


def test_a_recorded_function_runs_the_operators_again():
    """torch.jit.trace records the four operators: run on other inputs, the recorded function gives what the eager calls give and
    writes its caches."""
    hq, hk, dim, win, sinks, dtype = 4, 2, 64, 24, 2, torch.bfloat16
    freqs = torch.rand(dim // 2, generator=_gen(61)).to(DEV)
    pos, lengths, zero = torch.arange(47, device=DEV).view(47, 1), torch.tensor([30, 17], device=DEV), torch.tensor([0, 0], device=DEV)

    def run(q, k, v, cu, kc, vc):
        q, k = ops.rotary_embed(q, k, pos, freqs, [dim // 2])
        out = ops.attn_window(q, k, v, cu, win, sinks)
        ops.window_cache_append(k, v, cu, zero, kc, vc, sinks)
        return out, ops.attn_window_step(q[:2], k[:2], v[:2], lengths, kc, vc, sinks)

    def inputs(seed):
        q, k, v, cu, _, _ = _case([30, 17], None, hq, hk, dim, dtype, False, seed=seed)
        cache = [torch.zeros(2, hk, win + sinks, dim, dtype=dtype, device=DEV) for _ in range(2)]
        return tuple(_dev(q, k, v, cu)) + tuple(cache)

    again = torch.jit.trace(run, inputs(60), check_trace=False)
    kinds = [n.kind() for n in again.graph.nodes()]
    assert all('qcnet_hip::' + name in kinds for name in ops.SEQUENCE_OP_NAMES), kinds
    for seed in (62, 63):
        a, b = inputs(seed), inputs(seed)
        want, got = run(*a), again(*b)
        assert all(torch.equal(x, y) for x, y in zip(got + b, want + a))


def test_function_transforms_see_the_operators():
    """vmap over a batch equals the loop where the dispatcher can loop (an operator that returns one tensor) and is refused as an
    operator without a batching rule where it cannot; dual numbers reach the operator, which has no forward derivative."""
    g = _gen(64)
    q, k, v = (_rand(g, 3, 10, 2, 16).to(DEV) for _ in range(3))
    cu = torch.tensor([0, 4, 10], device=DEV)
    attend = lambda q, k, v: ops.attn_window(q, k, v, cu, 3, 1)
    assert torch.equal(torch.vmap(attend)(q, k, v), torch.stack([attend(*x) for x in zip(q, k, v)]))
    pos, freqs = torch.arange(10, device=DEV).view(10, 1), torch.rand(8, generator=g).to(DEV)
    with pytest.raises(RuntimeError, match='Batching rule not implemented for qcnet_hip::rotary_embed'):
        torch.vmap(lambda t: ops.rotary_embed(t, None, pos, freqs, [8])[0])(q)
    with torch.autograd.forward_ad.dual_level():
        got = attend(torch.autograd.forward_ad.make_dual(q[0], q[1]), k[0], v[0])
        assert torch.equal(torch.autograd.forward_ad.unpack_dual(got).primal, attend(q[0], k[0], v[0]))


# ------------------------------------------------------------------------------------------------
# weights of the 16-bit types
# ------------------------------------------------------------------------------------------------
HALVES = [torch.bfloat16, torch.float16]


def _full_tolerance(dtype, dim, r, v_max):
    """tolerance() of a form whose weights meet V as the sum of two numbers of the type.  With h half a step of the type, the rest of a
    weight p after its rounding is at most h p, and that is rounded by at most h of itself: h^2 p is lost; float16 also loses up to half
    of its smallest step (2^-25) of a rest, p relative to a sum of at least 1.  The output's rounding is the only one of size h."""
    o, mag, reach, count = r
    h = torch.finfo(dtype).eps / 2
    tol = ref.tolerance(torch.float32, dim, *r, v_max) + h * o.abs() * 1.01 + h * h * 1.01 * mag
    if dtype == torch.float16:
        tol = tol + (count.unsqueeze(-1) + 1) * 2.0 ** -25 * v_max
    return tol


@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('ages,hq,hk,dim,win,sinks', [([1, 5, 0, 30], 8, 8, 16, 50, 1), ([1, 300, 2], 8, 2, 64, 200, 4),
                                                      ([700, 1], 4, 1, 128, 600, 2), ([9000], 8, 1, 96, 2500, 0), ([3, 90], 3, 1, 32, 40, 0)])
def test_step_weights_keep_their_bits(ages, hq, hk, dim, win, sinks, dtype):
    q, k, v, lengths, kc, vc, km, mc = _step_case(ages, hq, hk, dim, win, sinks, False, dtype, seed=70)
    got = ops.attn_window_step(*_dev(q, k, v, lengths, kc, vc), sinks).cpu().double()
    r = ref.step(q, k, v, lengths, kc, vc, sinks)
    tol = _full_tolerance(dtype, dim, r, float(vc.double().abs().max()))
    assert bool(((got - r[0]).abs() <= tol).all()), float(((got - r[0]).abs() / tol).max())
    # a mean of equal values is that value: before the rounding it is off by h^2 (2^-16 or less) and by what float32 sums of at most about
    # 200 terms (one accumulator's) round, 2 x 200 x 2^-24, together less than 2^-14; half a step below 1 is 2^-9 or 2^-12
    one = torch.ones_like(v), torch.ones_like(vc)
    got = ops.attn_window_step(*_dev(q, k, one[0], lengths, kc, one[1]), sinks)
    assert bool((got == 1).all()), got[got != 1]


@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('lens,hq,hk,dim,win,sinks', [([59, 1, 0, 16], 8, 8, 16, 10, 1), ([200, 17], 4, 2, 8, 90, 2), ([70, 40], 6, 2, 24, 10, 3),
                                                      ([59, 30], 8, 8, 32, 16, 1), ([130], 7, 1, 16, 1000, 0)])
def test_window_weights_of_narrow_heads_keep_their_bits(lens, hq, hk, dim, win, sinks, dtype):
    q, k, v, cu, _, _ = _case(lens, None, hq, hk, dim, dtype, False, seed=71)
    got = ops.attn_window(*_dev(q, k, v, cu), win, sinks).cpu().double()
    r = ref.window(q, k, v, cu, win, sinks)
    tol = _full_tolerance(dtype, dim, r, float(v.double().abs().max()))
    assert bool(((got - r[0]).abs() <= tol).all()), float(((got - r[0]).abs() / tol).max())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lens,extra,hq,hk,dim,win,sinks', [
    ([59, 1, 0, 16], None, 8, 8, 16, 10, 1), ([150, 17], None, 4, 2, 16, 90, 2), ([59, 30], None, 8, 8, 32, 16, 1), ([59, 30], None, 8, 8, 32, 60, 1),
    ([150, 70], None, 4, 2, 64, 120, 2), ([90, 3], None, 4, 1, 128, 50, 0), ([20, 6], [2500, 1100], 2, 1, 64, 2200, 2)])
def test_window_weights_add_up_to_one(lens, extra, hq, hk, dim, win, sinks, dtype):
    """A mean of equal values is that value.  The sum is either of the rounded weights that V meets or V meets all but h^2 of them; the rest
    is what float32 sums of at most 700 terms (one part's, of the longest case) round, 2 x 700 x 2^-24 = 2^-13.5.  Half a step below 1 is
    2^-9 or 2^-12 in 16 bits; float32 shows the rounding itself."""
    q, k, v, cu_q, cu_k, _ = _case(lens, extra, hq, hk, dim, dtype, False, seed=72)
    got = ops.attn_window(*_dev(q, k, torch.ones_like(v), cu_q), win, sinks, cu_k=None if extra is None else cu_k.to(DEV)).cpu().double()
    if dtype == torch.float32:
        assert float((got - 1).abs().max()) <= 2 * 2300 * 2.0 ** -24
    else:
        assert bool((got == 1).all()), got[got != 1]


@pytest.mark.parametrize('dtype', DTYPES)
def test_the_largest_scale(dtype):
    """Equal scores of 0 stay a plain mean at every scale that is taken."""
    q, k, v, cu, _, _ = _case([40, 9], None, 4, 2, 64, dtype, False, seed=73)
    q = torch.zeros_like(q)
    got = ops.attn_window(*_dev(q, k, v, cu), 12, 1, scale=2.35e38)
    _check(got, ref.window(q, k, v, cu, 12, 1), dtype, 64, v)
    _, _, _, lengths, kc, vc, _, _ = _step_case([30, 4], 4, 2, 64, 20, 1, False, dtype, seed=73)
    got = ops.attn_window_step(*_dev(q[:2], k[:2], v[:2], lengths, kc, vc), 1, scale=2.35e38)
    _check(got, ref.step(q[:2], k[:2], v[:2], lengths, kc, vc, 1), dtype, 64, vc)


def test_writing_a_cache_shows_in_what_autograd_saved_of_it():
    """A product of a cache with something trainable keeps the cache for its backward pass: appending or stepping in between is an error
    there, as with torch's own operations in place, and not another gradient.  Inference tensors, which keep no count, are written too."""
    def cache():
        return tuple(torch.ones(2, 1, 6, 16, device=DEV) for _ in range(2)) + (torch.ones(2, 6, dtype=torch.bool, device=DEV),)

    x, n, cu = torch.ones(2, 1, 16, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV), torch.tensor([0, 1, 2], device=DEV)
    calls = (lambda kc, vc, mc: ops.window_cache_append(x, x, cu, n, kc, vc, 1, mask_cache=mc),
             lambda kc, vc, mc: ops.attn_window_step(x, x, x, n, kc, vc, 1, mask_cache=mc))
    for call in calls:
        w = torch.ones(16, device=DEV, requires_grad=True)
        kc, vc, mc = cache()
        loss = (kc * w).sum() + (vc * w).sum()
        before = [t._version for t in (kc, vc, mc)]
        call(kc, vc, mc)
        assert all(t._version > b for t, b in zip((kc, vc, mc), before))
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            loss.backward()
        with torch.inference_mode():
            call(*cache())


@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('win,parts', [(1100, 2), (1700, 3), (2200, 4), (2700, 5), (3100, 6), (3600, 7), (4000, 8)])
@pytest.mark.parametrize('dim', [24, 128])
def test_window_split_into_every_number_of_parts(dim, win, parts, dtype):
    from tempenslearnagg_qcnet_amd import sequence_ops
    lens, extra, hq = [21, 6], [4000, 900], 3
    q, k, v, cu_q, cu_k, mask = _case(lens, extra, hq, hq, dim, dtype, True, seed=51)
    code = {torch.float16: 1, torch.bfloat16: 2}[dtype]
    assert sequence_ops._window_workspace(0, code, 2, 27, k.size(0), hq, hq, dim, win, 2) == 27 * hq * parts * (dim + 2) * 4
    got = ops.attn_window(*_dev(q, k, v, cu_q), win, 2, cu_k=cu_k.to(DEV), key_mask=mask.to(DEV))
    _check(got, ref.window(q, k, v, cu_q, win, 2, cu_k, mask), dtype, dim, v)


def test_two_threads_on_streams_of_their_own():
    """Prompts and steps from two threads at once, each on its own stream with its own caches, are what one thread gives."""
    import threading
    hq, hk, dim, win, sinks, dtype = 8, 2, 64, 2200, 2, torch.bfloat16
    q, k, v, cu_q, cu_k, mask = _case([20, 6], [2500, 1100], hq, hk, dim, dtype, True, seed=80)
    dq, dk, dv, dcq, dck, dm = _dev(q, k, v, cu_q, cu_k, mask)
    freqs, zero = torch.rand(dim // 2, generator=_gen(81)).to(DEV), torch.zeros(2, dtype=torch.int64, device=DEV)

    def work(turns):
        kc, vc = (torch.zeros(2, hk, win + sinks, dim, dtype=dtype, device=DEV) for _ in range(2))
        mc = torch.zeros(2, win + sinks, dtype=torch.bool, device=DEV)
        lengths = dck[1:] - dck[:-1]
        ops.window_cache_append(dk, dv, dck, zero, kc, vc, sinks, key_mask=dm, mask_cache=mc)
        outs = []
        for i in range(turns):
            outs.append(ops.attn_window(dq, dk, dv, dcq, win, sinks, cu_k=dck, key_mask=dm))
            a, b = ops.rotary_embed(dq[i:i + 2], dk[i:i + 2], lengths.view(2, 1), freqs, [dim // 2])
            outs.append(ops.attn_window_step(a, b, dv[i:i + 2], lengths, kc, vc, sinks, mask_cache=mc))
            lengths = lengths + 1
        return outs + [kc, vc, mc]

    want, got = work(8), [None, None]
    torch.cuda.synchronize()

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[i] = work(8)
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g in got:
        assert g is not None and len(g) == len(want) and all(torch.equal(x, y) for x, y in zip(g, want))


@pytest.mark.parametrize('dtype', DTYPES)
def test_a_cache_row_is_taken_over_by_another(dtype):
    """The tokens of one row, as a view of the cache, appended to another row of the same cache; both then go on by themselves."""
    hk, hq, dim, win, sinks, n = 2, 4, 64, 30, 2, 25
    q, k, v, lengths, kc, vc, _, _ = _step_case([n, 0, 9], hq, hk, dim, win, sinks, False, dtype, seed=90)
    dk, dv = kc.to(DEV), vc.to(DEV)
    ops.window_cache_append(dk[0, :, :n].transpose(0, 1), dv[0, :, :n].transpose(0, 1), torch.tensor([0, 0, n, n], device=DEV),
                            torch.tensor([n, 0, 9], device=DEV), dk, dv, sinks)
    kc[1, :, :n], vc[1, :, :n] = kc[0, :, :n], vc[0, :, :n]
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)
    lengths[1] = n
    got = ops.attn_window_step(*_dev(q, k, v, lengths), dk, dv, sinks)
    _check(got, ref.step(q, k, v, lengths, kc, vc, sinks), dtype, dim, vc)
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)


# ------------------------------------------------------------------------------------------------
# values that are not finite
# ------------------------------------------------------------------------------------------------
FORMS = [
    # lens, extra keys, hq, hk, dim, window, sinks: every form of the window attention, and rows that end inside its width
    ([59, 1, 0, 16], None, 8, 8, 16, 10, 1), ([150, 70], None, 4, 2, 16, 90, 2), ([70, 40], None, 6, 2, 24, 10, 3),
    ([150, 70], None, 4, 2, 32, 60, 1), ([150, 70], None, 4, 2, 40, 60, 1), ([150, 300], None, 4, 2, 64, 100, 2),
    ([130, 31], None, 4, 1, 80, 50, 1), ([130], None, 3, 3, 96, 40, 0), ([150, 70], None, 4, 1, 128, 60, 2),
    ([20, 6], [2500, 1100], 2, 1, 64, 2200, 2), ([9], [4000], 3, 1, 72, 3600, 0),
]


def _same_kind(got, want, tol):
    """NaN where it is NaN, an infinity of the same sign where it is one, near where it is finite."""
    assert bool((got.isnan() == want.isnan()).all()), (got.isnan() != want.isnan()).nonzero()[:4]
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and bool((got.isinf() == inf).all())
    fine = torch.isfinite(want)
    assert bool(((got - want).abs() <= tol)[fine].all()), float(((got - want).abs() / tol)[fine].max())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('form', range(len(FORMS)))
def test_values_that_are_not_finite_reach_the_rows_that_see_them(form, dtype):
    """Single features of some keys are NaN or infinite, masked keys are NaN throughout: each element of each row is what the sum over
    the keys that the row sees makes it, in float64."""
    lens, extra, hq, hk, dim, win, sinks = FORMS[form]
    q, k, v, cu_q, cu_k, mask = _case(lens, extra, hq, hk, dim, dtype, True, seed=100 + form)
    g = _gen(101 + form)
    fine = float(v.double().abs().max())
    tol = ref.tolerance(dtype, dim, *ref.window(q, k, v, cu_q, win, sinks, cu_k, mask), fine)
    vv = v.clone()
    for fill in (float('nan'), float('inf'), -float('inf')):
        hit = torch.rand(v.size(0), hk, 1, generator=g) < 0.04
        vv[(hit & (torch.rand(v.shape, generator=g) < 0.2))] = fill
    vv[0, 0, dim - 1] = float('inf')
    k, vv = k.clone(), vv.clone()
    k[~mask], vv[~mask] = float('nan'), float('nan')
    want = ref.window(q, torch.where(mask[:, None, None], k, torch.zeros_like(k)), vv, cu_q, win, sinks, cu_k, mask)[0]
    got = ops.attn_window(*_dev(q, k, vv, cu_q), win, sinks, cu_k=None if extra is None else cu_k.to(DEV), key_mask=mask.to(DEV))
    _same_kind(got.cpu().double(), want, tol)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('form', range(len(FORMS)))
def test_a_score_of_minus_infinity_counts_for_nothing(form, dtype):
    """A key whose first feature is -inf, against queries whose first is 1: its score is -inf and its weight 0, also where a row ends inside
    the width that the kernel works on.  Beside it, a value of another key is infinite, so that the rows are formed a second time."""
    lens, extra, hq, hk, dim, win, sinks = FORMS[form]
    q, k, v, cu_q, cu_k, mask = _case(lens, extra, hq, hk, dim, dtype, True, seed=120 + form)
    at = int(cu_q[1] if extra is None else cu_k[1]) - 2
    mask[at - 1:at + 1] = True
    q, k, vv = q.clone(), k.clone(), v.clone()
    q[..., 0] = 1
    k[at, :, 0] = -float('inf')
    vv[at - 1, :, dim // 2] = float('inf')
    rest = mask.clone()
    rest[at] = False
    kk = k.clone()
    kk[at] = 0
    tol = ref.tolerance(dtype, dim, *ref.window(q, kk, v, cu_q, win, sinks, cu_k, rest), float(v.double().abs().max()))
    for values in (v, vv):
        want = ref.window(q, kk, values, cu_q, win, sinks, cu_k, rest)[0]
        got = ops.attn_window(*_dev(q, k, values, cu_q), win, sinks, cu_k=None if extra is None else cu_k.to(DEV), key_mask=mask.to(DEV))
        _same_kind(got.cpu().double(), want, tol)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('form', range(len(FORMS)))
def test_means_of_values_near_the_largest_float(form, dtype):
    """Values of 1e38 to 3e38: their sums are no floats, their means are."""
    lens, extra, hq, hk, dim, win, sinks = FORMS[form]
    q, k, v, cu_q, cu_k, _ = _case(lens, extra, hq, hk, dim, dtype, False, seed=140 + form)
    v = ((torch.rand(v.shape, generator=_gen(141)) + 0.5) * 2e38).to(dtype)
    r = ref.window(q, k, v, cu_q, win, sinks, cu_k)
    got = ops.attn_window(*_dev(q, k, v, cu_q), win, sinks, cu_k=None if extra is None else cu_k.to(DEV)).cpu().double()
    assert bool(((got - r[0]).abs() <= ref.tolerance(dtype, dim, *r, float(v.double().abs().max()))).all())


@pytest.mark.parametrize('lens,extra,hq,hk,dim,win,dtype', [
    ([4096], None, 8, 2, 128, 1024, torch.bfloat16), ([4096], None, 8, 8, 32, 1024, torch.float16), ([200, 333], [3000, 3000], 8, 2, 64, 3000, torch.bfloat16),
    ([700] * 4, None, 4, 4, 64, 500, torch.float32), ([700] * 4, None, 8, 8, 16, 500, torch.float32)])
def test_a_value_that_is_not_finite_does_not_cost_hundreds_of_calls(lens, extra, hq, hk, dim, win, dtype):
    """An infinite value that every row sees, queries that are NaN, values that are NaN throughout: a second pass over the keys at most, three
    to five times the call (a bound of 30 leaves room for a busy card)."""
    q, k, v, cu_q, cu_k, _ = _case(lens, extra, hq, hk, dim, dtype, False, seed=160)
    q, k, v, cu_q, cu_k = _dev(q, k, v, cu_q, cu_k)
    sink, gone = v.clone(), torch.full_like(v, float('nan'))
    sink[(cu_q if extra is None else cu_k)[:-1]] = float('inf')

    def time(q, v):
        times = []
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.attn_window(q, k, v, cu_q, win, 1, cu_k=cu_k)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[3]

    plain = time(q, v)
    for args in ((q, sink), (torch.full_like(q, float('nan')), v), (q, gone)):
        assert time(*args) < 30 * plain


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('case', range(len(STEPS)))
def test_step_values_that_are_not_finite(case, dtype):
    """Single features of some slots and of the new token are NaN or infinite: infinities of one sign stay what they are, both signs or a NaN
    among a feature's seen values make NaN, and the other features stay near."""
    ages, hq, hk, dim, win, sinks, masked = STEPS[case]
    q, k, v, lengths, kc, vc, km, mc = _step_case(ages, hq, hk, dim, win, sinks, masked, dtype, seed=170)
    clone = lambda t: None if t is None else t.clone()
    r = ref.step(q, k, v, lengths, kc.clone(), vc.clone(), sinks, km, clone(mc))
    tol = ref.tolerance(dtype, dim, *r, float(vc.double().abs().max()))
    g = _gen(171 + case)
    for fill in (float('nan'), float('inf'), -float('inf')):
        vc[(torch.rand(vc.shape, generator=g) < 1.2 / vc.size(2))] = fill
        v[(torch.rand(v.shape, generator=g) < 0.1)] = fill
    got = ops.attn_window_step(*_dev(q, k, v, lengths, kc, vc), sinks, key_mask=None if km is None else km.to(DEV),
                               mask_cache=None if mc is None else mc.to(DEV))
    want = ref.step(q, k, v, lengths, kc, vc, sinks, km, mc)[0]
    assert bool(want.isinf().any()) and bool(torch.isfinite(want).any())
    _same_kind(got.cpu().double(), want, tol)
