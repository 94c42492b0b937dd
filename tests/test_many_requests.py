"""Requests of one batch that share prompts and weights and differ in the rest: forked sequences, compacted pages, adapters, settings of their own --
through the models of every design and the batch engine."""
import random

import numpy as np
import pytest
import torch

import fidizen_helpers
import potosun_helpers
import seqmix_helpers
import tomopel_helpers
import tutunex_helpers
import zusuvik_helpers
from seqmix_helpers import rel_err, tokens
from test_request_sampling import plain

HELPERS = {"gitopel": seqmix_helpers, "fidizen": fidizen_helpers, "tomopel": tomopel_helpers, "zusuvik": zusuvik_helpers, "tutunex": tutunex_helpers,
           "potosun": potosun_helpers}
FAMILIES = [(f, "mixed") for f in HELPERS] + [("gitopel", "wide_pool"), ("fidizen", "odd"), ("tomopel", "odd"), ("tutunex", "wide")]
# fp32 models: rounding of 2^-24 per sum, some tens of them in a row; the same text run in steps of other sizes sums in other orders
TOL = 1e-4


def build(family, config, page=4, batch=8, **kw):
    h = HELPERS[family]
    return h.build(h.CONFIGS[config], torch.float32, page=page, batch=batch, **kw)[0]


def last_logits(m, seq, ids):
    return m.forward_batch([(seq, ids)]).clone()


@pytest.mark.gpu
@pytest.mark.parametrize("family,config", FAMILIES)
@pytest.mark.parametrize("length", [1, 7, 8, 37])
def test_forked_sequences_go_on_as_their_parent_would(family, config, length):
    m = build(family, config)
    V, text = m.config.vocab_size, None
    text = tokens(length, V, length)
    m.open("parent")
    last_logits(m, "parent", text)
    free = len(m.kv_cache.free_pages)
    m.kv_cache.fork("parent", ["a", "b"])
    assert len(m.kv_cache.free_pages) == free - (2 if length % 4 else 0) and m.kv_cache.length("b") == length
    m.kv_cache.close("parent")
    tails = {"a": tokens(9, V, 1), "b": tokens(5, V, 2)}
    got = {}
    for k in range(9):                                        # both go on, token by token, in one batch while both have some
        parts = [(s, [t[k]]) for s, t in tails.items() if k < len(t)]
        out = m.forward_batch(parts).clone()
        for (s, _), row in zip(parts, out):
            got[s] = row
    for s, t in tails.items():
        m.open("whole")
        want = last_logits(m, "whole", text + t)
        m.close("whole")
        assert rel_err(got[s][None], want) < TOL
    for s in tails:
        m.close(s)
    assert sorted(m.kv_cache.free_pages) == list(range(m.kv_cache.n_pages)) and not any(m.kv_cache.refs)


@pytest.mark.gpu
@pytest.mark.parametrize("family,config", FAMILIES)
def test_compacted_pages_hold_what_they_held(family, config):
    m, other = build(family, config), build(family, config)
    V = m.config.vocab_size
    for mm in (m, other):
        for s, n in (("a", 21), ("b", 9), ("c", 30), ("d", 4)):
            mm.open(s)
            last_logits(mm, s, tokens(n, V, n))
        mm.kv_cache.fork("c", ["e"])
        for s in ("a", "d"):
            mm.close(s)
    c = m.kv_cache
    held = {s: m.kv_cache.length(s) for s in c.seqs}
    rows = [c.token_rows(i, s, range(n)) for s, n in held.items() for i in range(len(c.kv))]
    n = c.compact()
    assert n == len({p for s in c.seqs.values() for p in s["pages"]}) and max(p for s in c.seqs.values() for p in s["pages"]) < n
    assert c.free_pages == list(range(c.n_pages - 1, n - 1, -1))
    for (k, v), (k2, v2) in zip(rows, [c.token_rows(i, s, range(held[s])) for s in held for i in range(len(c.kv))]):
        assert torch.equal(k, k2) and torch.equal(v, v2)
    for step in range(6):
        parts = [(s, [tokens(6, V, 50 + i)[step]]) for i, s in enumerate(held)]
        assert torch.equal(m.forward_batch(parts).clone(), other.forward_batch(parts).clone())
    assert c.compact() >= n


@pytest.mark.gpu
def test_fork_refuses_and_changes_nothing():
    m = build("gitopel", "mixed", batch=3, max_length=40, max_tokens=20)
    c = m.kv_cache
    m.open("a")
    last_logits(m, "a", [1, 2, 3, 4, 5])
    before = (list(c.free_pages), list(c.free_slots), {k: dict(v) for k, v in c.seqs.items()}, list(c.refs))
    for children, error in ((["a"], KeyError), (["b", "b"], KeyError), (["b", "c", "d"], RuntimeError)):
        with pytest.raises(error):
            c.fork("a", children)
    with pytest.raises(KeyError):
        c.fork("nobody", ["b"])
    m.open("long")
    last_logits(m, "long", tokens(4 * len(c.free_pages), 96, 1))
    with pytest.raises(RuntimeError):                         # a slot is left, a page is not
        c.fork("a", ["b"])
    c.close("long")
    assert c.fork("a", []) == []
    assert (sorted(c.free_pages), sorted(c.free_slots)) == (sorted(before[0]), sorted(before[1])) and c.seqs == before[2] and c.refs == before[3]
    # a sequence that holds nothing yet forks too
    m.open("empty")
    c.fork("empty", ["twin"])
    assert rel_err(last_logits(m, "twin", [5, 6]), last_logits(m, "empty", [5, 6])) < TOL


def adapters_for(m, seed, ranks=(3, 8)):
    """adapters beside products of layers whose tensors are their own, the last one without the first layer's"""
    g = torch.Generator().manual_seed(seed)
    shared = {ly.weights_of for ly in m.config.layers} | {i for i, ly in enumerate(m.config.layers) if ly.weights_of is not None}
    out = []
    for n, r in enumerate(ranks):
        a = {}
        for i in range(len(m.config.layers)):
            for what in ("proj", "out"):
                lin = getattr(m._layer_structs[i], what)
                if i in shared or (n == len(ranks) - 1 and i == 0 and what == "proj"):
                    continue
                a[i, what] = (torch.randn(r, lin.K, generator=g) * lin.K ** -0.5, torch.randn(lin.N, r, generator=g) * r ** -0.5, 0.3)
        out.append(a)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("family,config", FAMILIES)
def test_adapters_are_the_merged_weights(family, config):
    """prompts and single tokens of sequences with either adapter and with none, in one batch, against models with the products added to the weights"""
    m = build(family, config)
    V, ads = m.config.vocab_size, adapters_for(m, 5)
    m.load_adapters(ads)
    assert m.n_adapters == 2
    texts = {"none": tokens(19, V, 1), "first": tokens(23, V, 2), "second": tokens(5, V, 3), "again": tokens(23, V, 2)}
    named = {"none": None, "first": 0, "second": 1, "again": 0}
    for s, a in named.items():
        m.open(s, adapter=a)
    prompt = m.forward_batch([(s, t[:-2]) for s, t in texts.items()]).clone()
    m.kv_cache.fork("second", ["child"])                      # a child runs with its parent's
    steps = [m.forward_batch([(s, [t[len(t) - 2 + k]]) for s, t in texts.items()] + [("child", [texts["second"][3 + k]])]).clone() for k in range(2)]
    for i, (s, t) in enumerate(texts.items()):
        ref = build(family, config)
        if named[s] is not None:
            for (ly, what), (A, B, scale) in ads[named[s]].items():
                ref._tensors[ly][what + "_w"] += (scale * B.double() @ A.double()).float().cuda()
        ref.open("x")
        want = last_logits(ref, "x", t[:-2])
        assert rel_err(prompt[i:i + 1], want) < TOL
        for k in range(2):
            want = last_logits(ref, "x", [t[len(t) - 2 + k]])
            assert rel_err(steps[k][i:i + 1], want) < TOL
            if s == "second":
                assert rel_err(steps[k][4:5], want) < TOL
        if named[s] is not None:                              # (and they do something)
            plain_m = build(family, config)
            plain_m.open("x")
            assert rel_err(prompt[i:i + 1], last_logits(plain_m, "x", t[:-2])) > 1e-2
    with pytest.raises(RuntimeError):
        m.load_adapters([])
    m.clear()
    m.load_adapters([])
    with pytest.raises(ValueError):
        m.open("y", adapter=0)


@pytest.mark.gpu
def test_a_step_without_adapters_is_what_it_was():
    """bit by bit, beside loaded adapters that nobody names"""
    m, bare = build("tutunex", "mixed"), build("tutunex", "mixed")
    m.load_adapters(adapters_for(m, 1))
    for mm in (m, bare):
        mm.open("a"), mm.open("b")
    for parts in ([("a", tokens(20, 50, 1)), ("b", tokens(3, 50, 2))], [("a", [4]), ("b", [7])]):
        assert torch.equal(m.forward_batch(parts).clone(), bare.forward_batch(parts).clone())
    lin = m._layer_structs[0].proj
    m.clear()
    for bad in ({(99, "proj"): (torch.zeros(2, lin.K), torch.zeros(lin.N, 2), 1.0)}, {(0, "proj"): (torch.zeros(2, lin.K + 1), torch.zeros(lin.N, 2), 1.0)},
                {(0, "head"): (torch.zeros(2, lin.K), torch.zeros(lin.N, 2), 1.0)}):
        with pytest.raises(ValueError):
            m.load_adapters([bad])


def engine(m, **kw):
    from umbrella_amd.speculation.batch_engine import BatchEngine
    from umbrella_amd.speculation.speculation_utils import IdTokenizer
    e = BatchEngine(target_model_obj=m, tokenizer=IdTokenizer(), device="cuda:0", **kw)
    e.initialize()
    e.eos_tokens = []
    return e


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["gitopel", "tomopel", "fidizen"])
def test_the_engine_with_all_of_it(family, monkeypatch):
    """prompts with several continuations, an adapter and settings each: every token drawn is the definition's on the logits of its step, and the logits of
    a continuation are those of its text run alone"""
    from umbrella_amd.speculation import batch_engine
    from umbrella_amd.speculation.batch_engine import Sampling
    m = build(family, "mixed")
    V = m.config.vocab_size
    m.load_adapters(adapters_for(m, 3))
    drawn = []
    inner = batch_engine.sample_rows

    def spy(logits, u, **kw):
        tok, prob = inner(logits, u, **kw)
        drawn.append((logits.cpu().clone(), u.cpu(), {k: v.cpu() for k, v in kw.items()}, tok.cpu()))
        return tok, prob
    monkeypatch.setattr(batch_engine, "sample_rows", spy)
    prompts = [tokens(13, V, 1), tokens(8, V, 2), tokens(5, V, 3)]
    settings = [Sampling(0.8, 20, 0.9, 0.02, seed=1), None, Sampling(1.2, 0, 0.95, 0.0, seed=2)]
    e = engine(m)
    out = e.generate_batch(prompts, 6, sampling=settings, n=2, adapters=[0, None, 1])
    assert [len(o) for p in out for o in p] == [6] * 6 and out[1][0] == out[1][1] and out[0][0] != out[0][1]
    assert not m.kv_cache.seqs and not any(m.kv_cache.refs) and sorted(m.kv_cache.free_pages) == list(range(m.kv_cache.n_pages))
    for logits, u, kw, tok in drawn:
        for r in range(logits.shape[0]):
            assert int(tok[r]) == plain(logits[r].numpy(), float(u[r]), float(kw["temperature"][r]), int(kw["top_k"][r]), float(kw["top_p"][r]), float(kw["min_p"][r]))[0]
    last = drawn[-1][0]
    for i, (p, ad) in enumerate(zip(prompts, (0, None, 1))):
        for k in range(2):
            m.open("alone", adapter=ad)
            assert rel_err(last[2 * i + k][None], last_logits(m, "alone", p + out[i][k][:-1])) < TOL
            m.close("alone")
    # the same seeds draw the same again, another one does not; settings that are the engine's draw as before
    assert engine(m).generate_batch(prompts, 6, sampling=settings, n=2, adapters=[0, None, 1]) == out
    settings[0].seed = 7
    assert engine(m).generate_batch(prompts, 6, sampling=settings, n=2, adapters=[0, None, 1])[0] != out[0]
    assert engine(m).generate_batch(prompts, 6) == [o[0] for o in engine(m).generate_batch(prompts, 6, n=2)]


@pytest.mark.gpu
def test_the_engine_admits_what_fits_and_refuses_the_rest():
    from umbrella_amd.speculation.batch_engine import Sampling
    m = build("gitopel", "mixed", batch=4, max_length=40, max_tokens=64)
    e = engine(m)
    a, b = e.submit([1, 2, 3], 5, n=3), e.submit([4, 5], 5, n=2)
    steps = 0
    while e.step():
        steps += 1
        assert len(e.running) <= 4
    assert all(len(e.finished[i].generated) == 5 for i in (a, (a, 1), (a, 2), b, (b, 1)))
    with pytest.raises(ValueError):
        e.submit([1], 5, n=5)
    with pytest.raises(ValueError):
        e.submit([1], 5, n=0)
    with pytest.raises(ValueError):
        e.submit([1], 5, adapter=0)
    with pytest.raises(ValueError):
        e.generate_batch([[1], [2]], 3, sampling=[None])
    api = [e.generate(input_ids=[1, 2, 3], max_new_tokens=12, temperature=1.5, topk=0, topp=1.0, min_p=0.001, seed=s)["generated_tokens"] for s in (3, 3, 4, None, None)]
    assert all(len(t) == 12 for t in api) and api[0] == api[1] and len(set(map(tuple, api))) == 4        # a seed's draws are the same whatever the request's number
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=2.0),
                dict(top_k=-1), dict(top_k=1 << 31)):
        with pytest.raises(ValueError):
            e.submit([1], 5, sampling=Sampling(**bad))
    assert not e.queue
    with pytest.raises(ValueError):
        engine(m, repetition_penalty=1.2).submit([1], 5, sampling=Sampling())
    assert len(engine(m, repetition_penalty=1.2, temperature=0.8).generate_batch([[1, 2]], 4, n=2)[0][1]) == 4
    m.open("holder")
    e.submit([1], 5, n=4)
    with pytest.raises(RuntimeError):
        e.step()


@pytest.mark.gpu
def test_continuations_differ_under_a_penalty_too():
    """the engine's own sampling with a repetition penalty: every continuation draws for itself, the first as if it were alone, and a seed draws the same again"""
    m = build("gitopel", "mixed", batch=4)
    kw = dict(repetition_penalty=1.2, temperature=1.5, topk=60, topp=1.0, seed=3)
    out = engine(m, **kw).generate_batch([[1, 2, 3]], 12, n=4)[0]
    assert [len(t) for t in out] == [12] * 4 and len(set(map(tuple, out))) == 4
    assert engine(m, **kw).generate_batch([[1, 2, 3]], 12, n=4)[0] == out
    assert engine(m, **kw).generate_batch([[1, 2, 3]], 12)[0] == out[0]
    assert engine(m, **{**kw, "seed": 4}).generate_batch([[1, 2, 3]], 12, n=4)[0] != out


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(temperature=0.0), dict(temperature=1.3, topk=20, topp=0.95), dict(temperature=1.3, topk=20, repetition_penalty=1.3)])
@pytest.mark.parametrize("place", [0, 1])
def test_requests_without_settings_do_not_feel_their_neighbours(kw, place):
    """what the engine's settings draw is the same beside requests with settings of their own, while they run and when they have ended"""
    from umbrella_amd.speculation.batch_engine import Sampling
    m = build("gitopel", "mixed", batch=4)

    def texts(sampling):
        e = engine(m, **kw)
        e.repetition_penalty, penalty = 1.0, e.repetition_penalty          # (a request with settings is taken while the engine has no penalty)
        each = [([1, 2, 3], 14, None), ([7, 8], 5, sampling), ([5, 4, 9, 9], 9, None)]
        each.insert(2 * place, each.pop(1))
        ids = [e.submit(p, n, sampling=s) for p, n, s in each]
        e.repetition_penalty = penalty
        while e.step():
            pass
        out = {tuple(p): e.finished[i].generated for (p, _, _), i in zip(each, ids)}
        assert [len(out[tuple(p)]) for p, n, _ in each] == [n for _, n, _ in each]
        return out
    without, beside = texts(None), texts(Sampling(0.7, 5, 0.9, 0.1, seed=2))
    assert all(without[p] == beside[p] for p in ((1, 2, 3), (5, 4, 9, 9)))


@pytest.mark.gpu
@pytest.mark.parametrize("step", [0, 1, 4])
@pytest.mark.parametrize("copies", [1, 2])
def test_a_request_without_a_token_ends_alone(step, copies, monkeypatch):
    """one request's logits are NaN in a step: it ends there with an error, and its neighbours draw what they draw beside one that ends there by itself"""
    from umbrella_amd.speculation.batch_engine import RequestError, Sampling
    m = build("gitopel", "mixed", batch=8)

    def texts(bad):
        e = engine(m, temperature=1.2, topk=20)
        inner, calls = e.run_step, [0]

        def run_step(entries, end=()):
            logits = inner(entries, end)
            if bad and calls[0] == step:
                for i, (rid, _, _) in enumerate(entries):
                    if rid in ("bad", ("bad", 1)):
                        logits[i] = float("nan")
            calls[0] += 1
            return logits
        monkeypatch.setattr(e, "run_step", run_step)
        own = Sampling(0.9, 30, 0.9, 0.01, seed=4)
        e.submit([1, 2, 3], 9, request_id="own", sampling=own)
        e.submit([8, 8], 9 if bad else step + 1, request_id="bad", sampling=own, n=copies)
        e.submit([4, 5, 6, 7], 11, request_id="engine's")
        while e.step():
            pass
        assert not m.kv_cache.seqs and not any(m.kv_cache.refs) and not e.running
        return e.finished
    got, want = texts(True), texts(False)
    for i in ("own", "engine's"):
        assert got[i].generated == want[i].generated and got[i].error is None
    for i in ["bad", ("bad", 1)][:copies]:
        assert got[i].error and got[i].generated == want[i].generated[:step]
    e = engine(m)
    monkeypatch.setattr(e, "run_step", lambda entries, inner=e.run_step: inner(entries) * float("nan"))
    with pytest.raises(RequestError) as err:
        e.generate_batch([[1, 2], [3]], 4, sampling=Sampling())
    assert err.value.outputs == [[], []] and not e.finished and not m.kv_cache.seqs


@pytest.mark.gpu
def test_settings_that_cannot_be_drawn_by_are_refused_before_a_step():
    from umbrella_amd._lib import UmbError
    m = build("gitopel", "mixed", batch=4)
    e, want = engine(m, temperature=1.0, topk=20), engine(m, temperature=1.0, topk=20).generate_batch([[1, 2, 3], [4]], 6)
    ids = [e.submit([1, 2, 3], 6), e.submit([4], 6)]
    for wrong in (0, 3):                                      # before the prompts, and in mid-text
        for _ in range(wrong):
            e.step()
        for name, value in (("topk", 0), ("topk", 2000), ("topp", 0.0)):
            good = getattr(e, name)
            setattr(e, name, value)
            if value != 2000:                                 # (more than the vocabulary: all of it)
                with pytest.raises(UmbError):
                    e.step()
            setattr(e, name, good)
    while e.step():
        pass
    assert [e.finished[i].generated for i in ids] == want


@pytest.mark.gpu
def test_a_request_that_does_not_fit_stands_in_nobodys_way():
    m = build("gitopel", "mixed", batch=4, max_length=60, max_tokens=64)
    want = engine(m).generate_batch([[4, 5]], 5)[0]
    for holds, bad in (([1, 2], dict(input_ids=[1, 2, 3], max_new_tokens=5, n=4)),               # three slots are left
                       (tokens(60, 96, 1), dict(input_ids=[1, 2, 3], max_new_tokens=50, n=1)),   # too few pages
                       (tokens(60, 96, 1), dict(input_ids=[1, 2, 3], max_new_tokens=20, n=3))):
        e = engine(m)
        m.open("holder")
        last_logits(m, "holder", holds)
        wrong, right = e.submit(**bad), e.submit([4, 5], 5)
        with pytest.raises(RuntimeError):
            e.step()
        while e.step():
            pass
        assert e.finished[right].generated == want and not e.queue
        for i in [wrong] + [(wrong, k) for k in range(1, bad["n"])]:
            assert e.finished[i].error and not e.finished[i].generated
        m.close("holder")
        assert not m.kv_cache.seqs
    # a single request waits for a slot
    for s in "abcd":
        m.open(s)
    e = engine(m)
    i = e.submit([4, 5], 5)
    assert not e.step() and list(e.queue)
    m.close("b")
    while e.step():
        pass
    assert e.finished[i].generated == want


@pytest.mark.gpu
@pytest.mark.parametrize("after", [0, 1, 2])
def test_queued_requests_do_not_run_with_adapters_that_they_did_not_name(after):
    """adapters loaded anew, fewer or as many, while a request that names one is queued: it ends with an error, the others run"""
    m = build("tutunex", "mixed", batch=4)
    V, e = m.config.vocab_size, engine(m)
    want = engine(m).generate_batch([tokens(4, V, 1)], 5)[0]
    m.load_adapters(adapters_for(m, 5))
    first, named, last = e.submit(tokens(4, V, 1), 5), e.submit(tokens(4, V, 1), 5, n=2, adapter=1), e.submit(tokens(4, V, 1), 5)
    m.load_adapters(adapters_for(m, 6)[:after])
    while e.step():
        pass
    assert e.finished[first].generated == e.finished[last].generated == want
    for i in (named, (named, 1)):
        assert e.finished[i].error and not e.finished[i].generated
    assert not m.kv_cache.seqs and not e.queue
    if after:
        e.submit(tokens(4, V, 1), 5, request_id="new", adapter=after - 1)
        while e.step():
            pass
        assert len(e.finished["new"].generated) == 5
        e.submit(tokens(4, V, 1), 5, request_id="alone", adapter=0)
        m.load_adapters([])
        assert not e.step() and e.finished["alone"].error


@pytest.mark.gpu
def test_api_requests_with_min_p_are_answered_whatever_the_engine_runs_by():
    m = build("gitopel", "mixed", batch=4)
    ask = dict(input_ids=[1, 2, 3], max_new_tokens=8)
    for kw in (dict(repetition_penalty=1.3, temperature=0.0), dict(repetition_penalty=1.3, temperature=1.2, topk=20), dict(temperature=0.0, topk=-1, topp=1.5)):
        want = engine(m, **kw).generate(**ask)["generated_tokens"] if kw.get("topk", 1) > 0 else engine(m, temperature=0.0).generate(**ask)["generated_tokens"]
        for min_p in (0.0, 0.1):
            assert engine(m, **kw).generate(**ask, min_p=min_p)["generated_tokens"] == want
        *_, (text, _) = engine(m, **kw).generate_stream(**ask, min_p=0.1)
        assert text.split() == [str(t) for t in want]
    # a top-p above 1 keeps all, as it does without min_p; settings that are none are refused still
    e = engine(m, temperature=1.2, topk=0, topp=1.5)
    assert e.generate(**ask, min_p=0.05, seed=3)["generated_tokens"] == e.generate(**ask, topp=1.0, min_p=0.05, seed=3)["generated_tokens"]
    for bad in (dict(min_p=-0.1), dict(min_p=1.5), dict(min_p=float("nan")), dict(min_p=0.1, topk=-1)):
        with pytest.raises(ValueError):
            engine(m, temperature=1.2).generate(**ask, **bad)


def test_forks_and_pages_on_the_host(monkeypatch):
    """the bookkeeping alone: random forks, extensions and closings, every page held as often as it is listed"""
    from umbrella_amd.attn import cache as C
    monkeypatch.setattr(C, "copy_pages", lambda *a, **kw: None)
    c = C.PagedSeqCache([(1, 8, 0)], [(1, 2, 2)], 200, 12, "cpu", torch.float32, page=4)
    rng, names = random.Random(1), iter(range(10000))
    for _ in range(600):
        held = list(c.seqs)
        move = rng.random()
        if move < 0.25 and c.free_slots:
            c.open(next(names))
        elif move < 0.5 and held:
            s, n = rng.choice(held), rng.randint(1, 9)
            if c.can_extend(s, n):
                c.extend(s, n)
        elif move < 0.7 and held:
            s, n = rng.choice(held), rng.randint(0, 3)
            if n <= len(c.free_slots) and (c.length(s) % 4 == 0 or n <= len(c.free_pages)):
                kids = [next(names) for _ in range(n)]
                c.fork(s, kids)
                full = c.length(s) // 4
                for k in kids:
                    assert c.seqs[k]["pages"][:full] == c.seqs[s]["pages"][:full] and not set(c.seqs[k]["pages"][full:]) & set(c.seqs[s]["pages"])
        elif move < 0.95 and held:
            c.close(rng.choice(held))
        else:
            c.compact()
        listed = np.bincount([p for s in c.seqs.values() for p in s["pages"]], minlength=c.n_pages).tolist()
        assert c.refs == listed and sorted(c.free_pages) == [p for p in range(c.n_pages) if listed[p] == 0]
        for s in c.seqs.values():
            assert len(s["pages"]) == -(-s["len"] // 4) and len(set(s["pages"])) == len(s["pages"])
            if "cpu" == c.device and s["len"]:
                assert all(0 <= p < c.n_pages for p in s["pages"])
