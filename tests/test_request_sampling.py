"""Tokens drawn with settings per request (speculation/sampling.py, umb_sample_requests) against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from umbrella_amd import _lib
from umbrella_amd.speculation.sampling import MAX_VOCAB, sample_rows

EINVAL, AT = -22, 1 << 20
INF, NAN, LOWEST = float("inf"), float("nan"), torch.finfo(torch.float32).min


def plain(x, u, t, k, p, m):
    """(token, share of the kept mass) of one row, settings as float32 numbers; everything in 64 bits"""
    x = np.where(np.isnan(x), -INF, x).astype(np.float64)
    order = np.lexsort((np.arange(x.size), -x))
    order = order[x[order] > -INF]
    if not order.size:
        return -1, 0.0
    if not t > 0:
        return int(order[0]), 1.0
    v, w = x[order], np.ones(order.size)
    low = v < v[0]
    w[low] = np.exp((v[low] - v[0]) / t) if v[0] < INF else 0.0          # infinite ones share all mass, at any temperature
    first_k = w[:k] if 0 < k < x.size else w
    upto = np.cumsum(first_k)
    front = np.concatenate([[0.0], upto[:-1]])
    n = first_k.size
    if p < 1:
        n = min(n, max(1, int((front < p * upto[-1]).sum())))
    if m == m:
        n = min(n, max(1, int((first_k >= m).sum())))
    mass = upto[n - 1]
    u = min(max(u, 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    at = min(int((upto[:n] <= u * mass).sum()), n - 1)
    return int(order[at]), float(first_k[at] / mass)


def check(x, u, t, k, p, m, got=None):
    """x [rows, V] and a number per row of each: drawn on the device and by the definition.  A border between two tokens is off by some 1e-12 of the mass, so
    tokens are equal; shares are rounded to fp32 once, half a step of 2^-23, and their sums are good to 1e-11"""
    dev = "cuda:0"
    f = [torch.tensor(v, dtype=torch.float32) for v in (u, t, p, m)]
    ks = torch.tensor(k, dtype=torch.int32)
    tok, prob = got or sample_rows(x.to(dev), f[0].to(dev), temperature=f[1].to(dev), top_k=ks.to(dev), top_p=f[2].to(dev), min_p=f[3].to(dev))
    rows = [plain(x[r].cpu().numpy(), *(float(f[i][r]) for i in (0, 1)), int(ks[r]), *(float(f[i][r]) for i in (2, 3))) for r in range(x.shape[0])]
    assert tok.tolist() == [a for a, _ in rows]
    want = torch.tensor([b for _, b in rows], dtype=torch.float64)
    assert bool(((prob.cpu().double() - want).abs() <= want * (2.0 ** -24 + 1e-10)).all())


def draws(rows, seed):
    g = torch.Generator().manual_seed(seed)
    r = torch.rand(5, rows, generator=g)
    pick = torch.arange(rows) % 7
    k = torch.where((pick == 1) | (pick == 4), (1 + r[0] * 80).to(torch.int32), torch.zeros(rows, dtype=torch.int32))
    k = torch.where(pick == 6, 1 << 30, k)
    return dict(u=r[1].tolist(), t=torch.where(pick == 0, 0.0, 0.3 + 1.5 * r[2]).tolist(), k=k.tolist(),
                p=torch.where((pick == 2) | (pick == 4), 0.5 + 0.49 * r[3], torch.ones(rows)).tolist(), m=torch.where((pick == 3) | (pick == 4), 0.2 * r[4], torch.zeros(rows)).tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 1000, 1025, 4099, 32000, 128256])
@pytest.mark.parametrize("spread", [0.5, 2.0, 6.0])
def test_every_setting(V, spread):
    rows = 35
    x = torch.randn(rows, V, generator=torch.Generator().manual_seed(V)) * spread
    check(x, **draws(rows, V + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V", [(1, 151936), (130, 5000), (300, 777), (2, 524288), (9, 1024), (9, 1025), (9, 8192), (9, 8193), (9, 16384), (9, 16385), (66, 20001), (66, 32768),
                                    (65, 32769)])
def test_rows_and_vocabularies(rows, V):
    x = torch.randn(rows, V, generator=torch.Generator().manual_seed(rows)) * 3
    check(x, **draws(rows, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [5, 640, 40000])
def test_equal_logits(V):
    """ties go to the lower index: the sums are whole numbers, so every border is exact"""
    us = [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24]
    n = len(us)
    check(torch.full((n, V), -3.25), us, [0.7] * n, [0] * n, [1.0] * n, [0.0] * n)
    check(torch.full((n, V), 7.0), us, [0.7] * n, [4] * n, [1.0] * n, [0.0] * n)
    check(torch.full((n, V), LOWEST), us, [1.0] * n, [0] * n, [0.5] * n, [1.0] * n)
    check(torch.zeros(n, V) * -1.0, us, [0.0] * n, [0] * n, [1.0] * n, [0.0] * n)


@pytest.mark.gpu
def test_logits_of_few_values():
    """16-bit logits: hundreds of tokens share a value, and borders fall between them"""
    x = (torch.randn(28, 50000, generator=torch.Generator().manual_seed(3)) * 2).to(torch.bfloat16).float()
    check(x, **draws(28, 8))
    x = torch.randn(28, 50000, generator=torch.Generator().manual_seed(4)).round()
    check(x, **draws(28, 9))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [7, 3000, 40000])
def test_masks(V):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(14, V, generator=g) * 2
    x[0] = -INF                                   # nothing left
    x[1] = NAN
    x[2, 1:] = -INF                               # one token left
    x[3, :-1] = NAN
    x[4] = LOWEST                                 # the lowest finite value everywhere: tokens like any other
    x[5, ::2] = LOWEST
    x[6, ::2] = -INF
    x[7, 1::3] = NAN
    x[8, 2] = INF                                 # infinite logits take it all
    x[9, 2], x[9, 5] = INF, INF
    x[10, 2], x[10, 3] = INF, NAN
    x[11] = torch.where(torch.rand(V, generator=g) < 0.999, torch.tensor(-INF), x[11])
    x[11, V // 2] = 0.5
    x[12] *= 1e30                                 # far beyond what exp takes
    x[13] = x[13] * 1e-30
    for kw in (dict(k=0, p=1.0, m=0.0, t=1.0), dict(k=5, p=0.9, m=0.01, t=0.7), dict(k=0, p=1.0, m=0.0, t=0.0), dict(k=0, p=0.8, m=0.0, t=1e-30),
               dict(k=0, p=0.8, m=0.0, t=1e30), dict(k=0, p=0.95, m=0.0, t=INF)):
        for u in (0.0, 0.37, 0.99):
            check(x, [u] * 14, [kw["t"]] * 14, [kw["k"]] * 14, [kw["p"]] * 14, [kw["m"]] * 14)


@pytest.mark.gpu
def test_settings_at_their_ends():
    x = torch.randn(1, 3001, generator=torch.Generator().manual_seed(2)).repeat(12, 1) * 2
    u = [0.5, 1.0, 2.0, -1.0, NAN, 0.0, 0.999, 0.3, 0.3, 0.3, 0.3, 0.3]
    t = [1.0] * 9 + [NAN, -1.0, 0.5]
    k = [0, 10, 10, 10, 10, -5, 3001, 3002, 1, 0, 0, 3000]
    p = [0.0, 1.0, 1.0, 1.0, 1.0, 0.5, 2.0, NAN, 0.5, 1.0, 1.0, -1.0]
    m = [0.0, 0.0, 0.0, 0.0, 0.0, 2.0, 1.0, NAN, -1.0, 0.0, 0.0, 0.1]
    check(x, u, t, k, p, m)


@pytest.mark.gpu
def test_rows_apart_and_numbers_for_all():
    """rows of a wider matrix, at an odd address; one number for all rows; nothing beside the rows is touched"""
    wide = torch.randn(9, 1500, generator=torch.Generator().manual_seed(1)).cuda() * 2
    before = wide.clone()
    u = torch.rand(9, generator=torch.Generator().manual_seed(2))
    for lo, hi in ((3, 1203), (0, 1500), (1, 2)):
        got = sample_rows(wide[:, lo:hi], u.cuda(), temperature=0.8, top_k=20, top_p=0.9, min_p=0.01)
        check(wide[:, lo:hi].cpu(), u.tolist(), [0.8] * 9, [20] * 9, [0.9] * 9, [0.01] * 9, got=got)
    got = sample_rows(wide, u.cuda())
    check(wide.cpu(), u.tolist(), [1.0] * 9, [0] * 9, [1.0] * 9, [0.0] * 9, got=got)
    assert torch.equal(wide, before)
    tok, prob = sample_rows(wide[:0], u.cuda()[:0])
    assert tok.shape == (0,) and prob.shape == (0,)


@pytest.mark.gpu
def test_captured_and_on_streams():
    """a captured call replayed over new inputs, beside eager calls on another stream"""
    rows, V = 12, 20000
    s = draws(rows, 3)
    x, u = torch.zeros(rows, V, device="cuda:0"), torch.zeros(rows, device="cuda:0")
    kw = dict(temperature=torch.tensor(s["t"]).cuda(), top_k=torch.tensor(s["k"], dtype=torch.int32).cuda(), top_p=torch.tensor(s["p"]).cuda(),
              min_p=torch.tensor(s["m"]).cuda())
    sample_rows(x, u, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with _lib.capturing(graph):
        got = sample_rows(x, u, **kw)
    side = torch.cuda.Stream()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        hx, hu = torch.randn(rows, V, generator=g) * 2, torch.rand(rows, generator=g)
        x.copy_(hx), u.copy_(hu)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = sample_rows(hx.cuda(), hu.cuda(), **kw)
        torch.cuda.synchronize()
        check(hx, hu.tolist(), s["t"], s["k"], s["p"], s["m"], got=got)
        check(hx, hu.tolist(), s["t"], s["k"], s["p"], s["m"], got=beside)


def test_refusals_of_the_wrapper():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    for kw in (dict(logits=x), dict(logits=x.double()), dict(logits=x[0])):
        with pytest.raises(ValueError):
            sample_rows(uniforms=u, **kw)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, u = torch.zeros(2, 8, device="cuda:0"), torch.zeros(2, device="cuda:0")
    for bad in (dict(logits=x.t()), dict(logits=x[:1].expand(2, 8)), dict(logits=x[:, :0]), dict(logits=x.half()), dict(logits=torch.zeros(1, MAX_VOCAB + 1, device="cuda:0"), uniforms=u[:1]),
                dict(uniforms=u[:1]), dict(uniforms=u.cpu()), dict(uniforms=None), dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:1]),
                dict(min_p=torch.zeros(4, device="cuda:0")[::2])):
        with pytest.raises(ValueError):
            sample_rows(**{"logits": x, "uniforms": u, **bad})


@pytest.mark.parametrize("kw", [dict(rows=0), dict(V=0), dict(V=MAX_VOCAB + 1, ld=MAX_VOCAB + 1), dict(ld=63), dict(logits=None), dict(tokens=None), dict(uniforms=None),
                                dict(scratch=None), dict(scratch=AT + 4), dict(scratch_bytes=0)])
def test_refusals_of_the_entry_point(kw):
    """before anything is launched: the addresses are never read"""
    a = dict(tokens=AT, logits=AT, ld=64, rows=3, V=64, uniforms=AT, scratch=AT, scratch_bytes=None)
    a.update(kw)
    lib = _lib.load_seq()
    n = lib.umb_sample_requests_bytes(3, 64) if a["scratch_bytes"] is None else a["scratch_bytes"]
    assert lib.umb_sample_requests_bytes(0, 64) == 0 and lib.umb_sample_requests_bytes(3, 0) == 0 and lib.umb_sample_requests_bytes(1, MAX_VOCAB + 1) == 0
    assert lib.umb_sample_requests(a["tokens"], None, a["logits"], a["ld"], a["rows"], a["V"], a["uniforms"], None, None, None, None, a["scratch"], n, None) == EINVAL


def check_finely(x, u, t, k, p, m):
    """check, with sums in 80 bits: in 64, half a million additions of 1e-11 to 1 are off by whole tokens themselves (2^-53 each, 524288 of them 6e-11: four tokens)"""
    got = sample_rows(x.cuda(), *(torch.tensor(v, dtype=torch.float32).cuda() for v in (u, t)), top_k=torch.tensor(k, dtype=torch.int32).cuda(),
                      top_p=torch.tensor(p, dtype=torch.float32).cuda(), min_p=torch.tensor(m, dtype=torch.float32).cuda())
    want, shares = [], []
    for r in range(x.shape[0]):
        v = x[r].numpy().astype(np.longdouble)
        order = np.lexsort((np.arange(v.size), -v))
        order = order[v[order] > -INF]
        w = np.exp((v[order] - v[order[0]]) / np.longdouble(np.float32(t[r])))
        w = w[:k[r]] if k[r] > 0 else w
        upto = np.cumsum(w)
        n = min(int((np.concatenate([[0.0], upto[:-1]]) < np.longdouble(np.float32(p[r])) * upto[-1]).sum()) if p[r] < 1 else w.size, int((w >= np.float32(m[r])).sum()))
        at = min(int((upto[:n] <= np.longdouble(np.float32(u[r])) * upto[n - 1]).sum()), n - 1)
        want.append(int(order[at])), shares.append(float(w[at] / upto[n - 1]))
    assert got[0].tolist() == want
    shares = torch.tensor(shares, dtype=torch.float64)
    assert bool(((got[1].cpu().double() - shares).abs() <= shares * (2.0 ** -24 + 1e-10)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("V,down", [(128256, 20.0), (262144, 18.0), (30000, 15.0), (524288, 25.0)])
def test_draws_from_equal_logits_far_below_one(V, down):
    """a share of 1e-4 and less in tokens of 1e-9 each: u counts them off"""
    x = torch.full((1, V), 3.0 - down)
    x[0, V // 3] = 3.0
    share = (V - 1) * np.exp(-down) / (1 + (V - 1) * np.exp(-down))
    u = [0.99975723] if V == 128256 else []
    u += [1.0 - share * f for f in np.linspace(0.01, 0.99, 40)]
    r = len(u)
    check_finely(x.expand(r, V).contiguous(), u, [1.0] * r, [0] * r, [1.0] * r, [0.0] * r)


@pytest.mark.gpu
@pytest.mark.parametrize("V,n,settings", [(1000, 999, ((0, 0.0), (1000, 0.0), (0, 1e-12))), (40000, 900, ((901, 0.0), (901, 1e-12))), (40000, 1500, ((0, 0.0), (1501, 0.0), (0, 1e-12)))])
def test_draws_from_few_logits_far_below_one(V, n, settings):
    """the same among tokens that are put in order, at every u that is in the tail"""
    x, u = [], []
    for i in range(0, 300, 1 if V < 2000 else 4):
        down = float(np.float32(21 + 0.01 * i))
        share = n * np.exp(-down) / (1 + n * np.exp(-down))
        row = torch.full((V,), -INF)
        row[V // 2 - n // 2:V // 2 - n // 2 + n + 1] = -down
        row[V // 2] = 0.0
        for k in range(1, 13):
            if k * 2.0 ** -24 < share:
                x.append(row), u.append(1.0 - k * 2.0 ** -24)
    x, r = torch.stack(x), len(u)
    for k, m in settings:
        check_finely(x, u, [1.0] * r, [k] * r, [1.0] * r, [m] * r)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [600, 1025, 8193, 20000, 40000, 128256])
def test_equal_logits_among_masked_ones(V):
    """n tokens of one value and nothing else: every share is a whole number of n-ths, and a p or u that is one too ends at the token that 64 bits end at"""
    g = torch.Generator().manual_seed(V)
    x, u, t, p = [], [], [], []
    for n in (2, 3, 4, 8, 100):
        for value, temperature in ((3.0, 1.0), (7.0, 0.7), (5.1, 1.0), (-2.3, 0.9)):
            row = torch.full((V,), -INF)
            row[torch.randperm(V, generator=g)[:n]] = value
            for share in (0.25, 0.5, 0.75):
                for uu, pp in ((share, 1.0), (0.6, share), (share, share)):
                    x.append(row), u.append(uu), t.append(temperature), p.append(pp)
    r = len(x)
    check(torch.stack(x), u, t, [0] * r, p, [0.0] * r)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1025, 40000, 128256])
@pytest.mark.parametrize("k", [0, 2, 100, 1000, 1025])
@pytest.mark.parametrize("rest,down", [(1000, 30.0), (1000, 25.0), (1 << 20, 34.0), (1 << 20, 60.0)])
def test_equal_logits_above_a_faint_tail(V, rest, down, k):
    """two and four largest, and tokens so far below that all of them together weigh some 1e-10 of the row: enough to say on which side of p the largest stand
    (60 down: too little even for 64 bits, whose sums are whole)"""
    g = torch.Generator().manual_seed(V)
    x, u, t, p = [], [], [], []
    for n in (2, 4):
        for value, temperature in ((3.0, 1.0), (7.0, 0.7), (5.1, 1.0), (-2.3, 0.9)):
            row = torch.full((V,), -INF)
            order = torch.randperm(V, generator=g)
            row[order[n:n + rest]] = value - down * temperature
            row[order[:n]] = value
            for share in (0.25, 0.5, 0.75):
                x.append(row), u.append(0.6), t.append(temperature), p.append(share)
    r = len(x)
    check(torch.stack(x), u, t, [k] * r, p, [0.0] * r)
