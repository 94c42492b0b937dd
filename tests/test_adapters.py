"""Low-rank adapters of many requests beside a shared product (models/adapters.py, umb_seq_adapters) against the formula in 64 bits."""
import pytest
import torch

from umbrella_amd import _lib
from umbrella_amd.models.adapters import add_adapters, stack_adapters

EINVAL, AT, OUT = -22, 1 << 20, 1 << 24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(T, K, N, S, R, dtype, seed=0, ids="runs", ranks=None, size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, K, generator=g) * size).to(dtype)
    a, b = (torch.randn(S, R, K, generator=g) * K ** -0.5).to(dtype), (torch.randn(S, N, R, generator=g) * 0.5).to(dtype)
    if ids == "runs":
        adapter = torch.randint(-1, S, (max(1, T // 5),), generator=g).repeat_interleave(5).repeat(2)[:T] if T >= 5 else torch.randint(0, S, (T,), generator=g)
    elif ids == "one":
        adapter = torch.full((T,), S - 1)
    else:
        adapter = torch.randint(-1, S, (T,), generator=g)
    assert adapter.numel() == T
    rank = None if ranks is None else torch.tensor([ranks[i % len(ranks)] for i in range(S)], dtype=torch.int32)
    return dict(base=torch.randn(T, N, generator=g), x=x, a=a, b=b, adapter=adapter.to(torch.int32), scale=0.5 + torch.rand(S, generator=g), rank=rank)


def plain(base, x, a, b, adapter, scale, rank):
    """the formula, and how far a result may be from it: sums of n products in fp32 are off by at most n 2^-24 of the sum of their sizes (twice that where
    the matrix pipe cuts instead of rounding); u's terms hold 2^-22 of the row's largest (fp16), 2^-24 of it otherwise"""
    T, K = x.shape
    S, R = a.shape[:2]
    out, tol, eps = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64), 2.0 ** -24
    for i in range(S):
        rows = (adapter == i).nonzero()[:, 0]
        r = R if rank is None else max(0, min(R, int(rank[i])))
        if not rows.numel() or not r:
            continue
        xs, A, B, s = x[rows].double(), a[i, :r].double(), b[i, :, :r].double(), 1.0 if scale is None else float(scale[i])
        u = s * xs @ A.t()
        size_u, most = abs(s) * xs.abs() @ A.abs().t(), u.abs().max(1, keepdim=True).values
        out[rows] += u @ B.t()
        held = most * (4 * eps if x.dtype == torch.float16 else eps)
        tol[rows] = ((2 * K + 40) * eps * size_u + 2 * held) @ B.abs().t() + (6 * r + 16) * eps * (u.abs() @ B.abs().t())
    return out, tol + 3 * eps * (out.abs() + base.double().abs())


def check(kw, inplace=False):
    want, tol = plain(**kw)
    dev = {k: None if v is None else v.cuda() for k, v in kw.items()}
    got = add_adapters(**dev, out=dev["base"] if inplace else None)
    assert got.dtype == torch.float32 and (got is dev["base"]) == inplace
    if not inplace:
        assert torch.equal(dev["base"].cpu(), kw["base"])
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    none = (kw["adapter"] < 0) | (kw["adapter"] >= kw["a"].shape[0])
    assert torch.equal(got.cpu()[none], kw["base"][none])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 130])
@pytest.mark.parametrize("ids", ["runs", "any", "one"])
def test_rows(name, T, ids):
    check(make(T, 256, 192, 5, 16, TYPES[name], seed=T, ids=ids))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("R", [1, 3, 8, 10, 16, 17, 24, 32, 33, 64, 72, 100, 127, 128])
def test_ranks(name, R):
    check(make(37, 136, 84, 4, R, TYPES[name], seed=R, ids="any"))
    check(make(80, 136, 84, 2, R, TYPES[name], seed=R, ids="any", ranks=[max(1, R // 3), R]))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("T", [1, 40, 200, 300])
def test_ranks_that_end_in_every_tile(name, T):
    """Products of tiles of 16 ranks, of which some adapters have all, some a few of the last and some none: with a branch between two of them, the last sum of four was
    read before it was there (rank 72: of 67 and 71)"""
    for R in (32, 64, 128):
        check(make(T, 264, 84, 8, R, TYPES[name], seed=T + R, ids="any", ranks=[R, R // 2 + 8, R // 2 + 1, R - 7, R - 15, 9, 24, R - 16]))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("K,N", [(1, 1), (7, 5), (8, 4), (31, 66), (33, 255), (40, 256), (100, 257), (184, 520), (1000, 1030), (4096, 300), (264, 5000)])
def test_widths(name, K, N):
    check(make(19, K, N, 3, 8, TYPES[name], seed=K, ids="any"))
    check(make(70, K, N, 3, 16, TYPES[name], seed=K, ids="runs"))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("R,K", [(8, 4096), (8, 4104), (16, 2048), (32, 1024), (33, 990), (64, 512), (64, 520), (1, 32768), (1, 33000)])
@pytest.mark.parametrize("T", [1, 5, 64, 65])
def test_both_sides_of_one_launch(name, R, K, T):
    """the sizes up to which both products are one launch, and just beyond"""
    check(make(T, K, 300, 3, R, TYPES[name], seed=T, ids="any", ranks=[R, max(1, R - 3)]), inplace=T == 5)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [255, 256, 257, 511, 700, 1025, 2049])
@pytest.mark.parametrize("ids", ["runs", "any", "one"])
def test_more_rows_than_a_window(T, ids):
    check(make(T, 96, 72, 7, 24, torch.bfloat16, seed=T, ids=ids), inplace=ids == "any")


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
def test_one_long_prompt(name):
    check(make(3000, 512, 384, 2, 64, TYPES[name], ids="one"))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
def test_every_row_an_adapter_of_its_own(name):
    kw = make(200, 264, 136, 200, 16, TYPES[name])
    kw["adapter"] = torch.randperm(200, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    check(kw, inplace=True)


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("size", [1e-6, 1e4])
def test_small_and_large_inputs(name, size):
    """fp16: sums beyond its largest number, and below its smallest"""
    check(make(33, 512, 64, 3, 16, TYPES[name], ids="any", size=size))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
def test_numbers_that_are_no_adapter(name):
    kw = make(90, 64, 48, 4, 8, TYPES[name], ids="any")
    kw["adapter"][::3], kw["adapter"][1::7], kw["adapter"][5] = -1, 4, 1 << 30
    kw["adapter"][6] = -(1 << 31)
    check(kw)
    kw["adapter"][:] = -1
    check(kw)
    check(kw, inplace=True)


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("R", [16, 13])
def test_what_stands_behind_a_rank_is_not_read_into_anything(name, R):
    kw = make(50, 72, 100, 3, R, TYPES[name], ids="any", ranks=[5, 0, R])
    dirty = dict(kw, a=kw["a"].clone(), b=kw["b"].clone())
    for i, r in enumerate(kw["rank"].tolist()):
        dirty["a"][i, r:], dirty["b"][i, :, r:] = float("nan"), float("inf")
    got = check(kw)
    dev = {k: v.cuda() for k, v in dirty.items()}
    assert torch.equal(add_adapters(**dev), got)


@pytest.mark.gpu
def test_infinities_stay_in_their_rows():
    kw = make(40, 64, 48, 2, 8, torch.bfloat16, ids="any")
    clean = check(kw).cpu()
    kw["x"][3, 5], kw["x"][7, 2], kw["base"][9, 1] = float("inf"), float("nan"), float("inf")
    kw["adapter"][[3, 7]] = 1
    got = add_adapters(**{k: None if v is None else v.cuda() for k, v in kw.items()}).cpu()
    assert not got[7].isfinite().any() and not got[3].isfinite().any() and got[9, 1] == float("inf")
    others = [i for i in range(40) if i not in (3, 7, 9)]
    assert torch.equal(got[others], clean[others])


@pytest.mark.gpu
def test_addresses_of_odd_alignment():
    """operands that start 4 bytes (fp32) or 2 bytes (16 bits) into their memory"""
    kw = make(37, 64, 48, 3, 8, torch.float16, ids="any")

    def shifted(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda:0")
        flat[1:] = t.reshape(-1).cuda()
        return flat[1:].view(t.shape)
    want, tol = plain(**kw)
    dev = {k: None if v is None else (shifted(v) if k in ("base", "x", "a", "b") else v.cuda()) for k, v in kw.items()}
    assert bool(((add_adapters(**dev).cpu().double() - want).abs() <= tol).all())


@pytest.mark.gpu
def test_stacked_from_adapters_of_several_ranks():
    g = torch.Generator().manual_seed(4)
    each = [(torch.randn(r, 64, generator=g), torch.randn(48, r, generator=g), 0.25 * r) for r in (4, 9, 16)]
    a, b, scale, rank = stack_adapters(each, device="cuda:0", dtype=torch.bfloat16)
    assert a.shape == (3, 16, 64) and b.shape == (3, 48, 16) and rank.tolist() == [4, 9, 16]
    kw = make(21, 64, 48, 3, 16, torch.bfloat16, ids="any")
    kw.update(a=a.cpu(), b=b.cpu(), scale=scale.cpu(), rank=rank.cpu())
    got = check(kw)
    kw["rank"] = None                             # what is added to a rank is zeros
    assert torch.allclose(check(kw), got, rtol=0, atol=1e-4)


@pytest.mark.gpu
def test_captured_and_on_streams():
    kw = make(70, 256, 192, 5, 16, torch.bfloat16, ids="any")
    dev = {k: None if v is None else v.cuda() for k, v in kw.items()}
    add_adapters(**dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with _lib.capturing(graph):
        got = add_adapters(**dev)
    side = torch.cuda.Stream()
    for seed in range(3):
        new = make(70, 256, 192, 5, 16, torch.bfloat16, seed=seed + 9, ids="any")
        for k in ("base", "x", "a", "b", "adapter", "scale"):
            dev[k].copy_(new[k])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = add_adapters(**dev)
        torch.cuda.synchronize()
        want, tol = plain(**new)
        for t in (got, beside):
            assert bool(((t.cpu().double() - want).abs() <= tol).all())
        assert torch.equal(got, beside)


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("T", [257, 512, 700])
def test_as_many_adapters_as_rows(name, T):
    """every row of a window its own, in any order; the same bits again"""
    kw = make(T, 40, 36, 900, 8, TYPES[name], seed=T, ids="any", ranks=[8, 3, 0, 5])
    kw["adapter"] = torch.randperm(900, generator=torch.Generator().manual_seed(T))[:T].to(torch.int32)
    assert torch.equal(check(kw), check(kw))
    kw["adapter"][::3] = torch.tensor([-1, 1 << 30, -(1 << 31), 900])[torch.arange(len(kw["adapter"][::3])) % 4].to(torch.int32)
    check(kw)


def test_refusals_of_the_wrapper():
    kw = make(4, 16, 8, 2, 8, torch.float32)
    kw.pop("rank")
    with pytest.raises(ValueError):
        add_adapters(**kw)                        # not on a GPU
    with pytest.raises(ValueError):
        stack_adapters([])
    with pytest.raises(ValueError):
        stack_adapters([(torch.zeros(4, 8), torch.zeros(6, 4), 1.0), (torch.zeros(4, 9), torch.zeros(6, 4), 1.0)])
    with pytest.raises(ValueError):
        stack_adapters([(torch.zeros(129, 8), torch.zeros(6, 129), 1.0)])


@pytest.mark.gpu
def test_refusals_on_the_device():
    kw = {k: None if v is None else v.cuda() for k, v in make(4, 16, 8, 2, 8, torch.bfloat16).items()}
    bad = [dict(x=kw["x"].float()), dict(x=kw["x"][:3]), dict(a=kw["a"][:, :7]), dict(b=kw["b"][:, :7]), dict(base=kw["base"].half()), dict(adapter=kw["adapter"].long()),
           dict(adapter=kw["adapter"][:3]), dict(scale=kw["scale"][:1]), dict(rank=torch.zeros(2, device="cuda:0")), dict(out=kw["base"][:, :7]), dict(adapter=kw["adapter"].cpu()),
           dict(x=kw["x"].t().contiguous().t()), dict(out=kw["base"].double()), dict(x=kw["x"].double(), a=kw["a"].double(), b=kw["b"].double())]
    for b in bad:
        with pytest.raises(ValueError):
            add_adapters(**{**kw, **b})
    empty = {k: v[:0] if k in ("base", "x", "adapter") else v for k, v in kw.items()}
    assert add_adapters(**empty).shape == (0, 8)


@pytest.mark.parametrize("kw", [dict(T=0), dict(N=0), dict(K=0), dict(S=0), dict(R=0), dict(R=129), dict(out=None), dict(base=None), dict(x=None), dict(a=None), dict(b=None),
                                dict(adapter=None), dict(scratch=None), dict(scratch=AT + 4), dict(floats=-1), dict(dtype=3),
                                # out over what is read: the base but in part, the last byte of x, a, b
                                dict(base=OUT + 4), dict(base=OUT - 3199), dict(x=OUT), dict(x=OUT - 3199), dict(x=OUT + 3199), dict(a=OUT - 511), dict(b=OUT - 255)])
def test_refusals_of_the_entry_point(kw):
    a = dict(T=100, N=8, K=16, S=2, R=8, out=OUT, base=OUT, x=AT, a=AT, b=AT, adapter=AT, scratch=AT, floats=0, dtype=1)
    a.update(kw)
    lib = _lib.load_seq()
    n = lib.umb_seq_adapters_floats(100, 16, 8) + a["floats"]
    assert lib.umb_seq_adapters_floats(0, 8, 8) == 0 and lib.umb_seq_adapters_floats(8, 0, 8) == 0 and lib.umb_seq_adapters_floats(8, 8, 129) == 0
    assert lib.umb_seq_adapters_floats(100, 16, 8) > 0 and lib.umb_seq_adapters_floats(4, 16, 8) == 0        # few tokens: one launch, no scratch
    assert lib.umb_seq_adapters(a["out"], a["base"], a["x"], a["a"], a["b"], a["adapter"], None, None, a["T"], a["N"], a["K"], a["S"], a["R"], a["scratch"], n, a["dtype"],
                                None) == EINVAL
