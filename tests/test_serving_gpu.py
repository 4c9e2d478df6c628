"""The operators of a serving step together, as they are used: sessions whose pages are kept on the device, keys and values in 4 bits,
log probabilities of what comes out; sessions, graphs, scoring and the commands."""

import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import hybrid_models as hm
import veredra_models as vm
from oracle import hybrid as oh
from oracle import veredra as ov
from test_cache4_gpu import kept
from test_hybrid_gpu import ROOT, close
from test_logprobs_gpu import SUM, reference, same

pytestmark = pytest.mark.gpu
_cache = {}


def model(name, dtype, cache):
    if (name, dtype, cache) not in _cache:
        from bitexact_llm_b200.hybrid import veredra
        cfg = vm.CONFIGS[name]
        _cache[name, dtype, cache] = veredra.load(cfg, vm.weights(cfg), "cuda", dtype, cache=cache)
    return _cache[name, dtype, cache]


def attention4(h, w, cfg, eps):
    """oracle.veredra.attention over the keys and values that the 4-bit cache keeps."""
    T, H, G, dk, dv, rot = h.shape[0], cfg["heads"], cfg["kv_heads"], cfg["dim"], cfg["vdim"], cfg["rot"]
    q = ov.rms_norm(ov.mat(h, w["q"]) + w["q.b"], w["q.norm"], eps).reshape(T, H, dk)
    k = ov.rms_norm(ov.mat(h, w["k"]) + w["k.b"], w["k.norm"], eps).reshape(T, G, dk)
    v = (ov.mat(h, w["v"]) + w["v.b"]).reshape(T, G, dv)
    q, k = ov.rotate_halves(q, rot["base"], rot["dims"]), ov.rotate_halves(k, rot["base"], rot["dims"])
    k, v = kept(torch.tensor(k)).numpy(), kept(torch.tensor(v)).numpy()
    own = np.arange(H) // (H // G)
    s = np.einsum("ihd,jhd->hij", q, k[:, own]) * cfg["scale"]
    p = ov.sink_softmax(s, ov.window_mask(T, (cfg.get("mask") or {}).get("size")), w["sink"])
    return ov.mat(np.einsum("hij,jhd->ihd", p, v[:, own]).reshape(T, H * dv), w["o"])


@pytest.mark.parametrize("name,n", [("one", 30), ("looped", 70), ("wide", 90)])
def test_model_with_a_4_bit_cache_against_the_oracle(name, n, monkeypatch):
    """32-bit: the whole model over keys and values as the definition keeps them."""
    from bitexact_llm_b200.decode import Session
    cfg, eng = vm.CONFIGS[name], model(name, "float32", "fp4")
    toks = np.random.RandomState(n).randint(0, cfg["vocab"], n).tolist()
    monkeypatch.setitem(ov.MIXERS, "attention", attention4)
    want = ov.forward(cfg, hm.as_numpy(vm.weights(cfg)), toks)[0]
    ses = Session(eng, 1, 128)
    x = torch.cat([ses.feed([(0, toks[a:b])])[0] for a, b in ((0, n // 2), (n // 2, n // 2 + 1), (n // 2 + 1, n))])
    close(eng.logits_float(x).cpu().numpy(), want, "float32")
    ses.check()


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
def test_portions_decoding_and_unequal_batches(dtype):
    """A prompt at once, in portions beside others, and token by token give the same model (to the rounding of its products: a key that is
    rounded the other way may get another code, so a position in ten may differ by more)."""
    from bitexact_llm_b200.decode import Session
    eng = model("wide", dtype, "fp4")
    toks = np.random.RandomState(1).randint(0, 300, 150).tolist()
    other = np.random.RandomState(2).randint(0, 300, 40).tolist()
    whole = eng.logits_float(Session(eng, 1, 256).feed([(0, toks)])[0]).double().cpu()
    ses = Session(eng, 3, 256, pages=12, on_device=True)
    rows = []
    for a, b in ((0, 1), (1, 70), (70, 71), (71, 148)):
        rows.append(ses.feed([(2, toks[a:b]), (0, other[a % 20:a % 20 + 3])])[0])
    for t in toks[148:]:
        active = torch.tensor([False, False, True]).cuda()
        rows.append(ses.step(torch.tensor([0, 0, t]).cuda(), active=active)[2:])
    got = eng.logits_float(torch.cat(rows)).double().cpu()
    assert ses.lens.tolist() == [12, 0, 150]
    err = ((got - whole) ** 2).mean(-1).sqrt() / (whole ** 2).mean().sqrt()
    assert (err > {"float32": 1e-3, "bfloat16": 0.08}[dtype]).float().mean() <= 0.1 and err.max() < 0.5, err.max()
    ses.check()


def test_cache_is_smaller_and_refused_where_there_is_none():
    from bitexact_llm_b200.hybrid import fedatar, veredra
    big, small = (model("wide", "bfloat16", c).new_cache(2, 9, 64) for c in (None, "fp4"))
    sizes = [sum(t.numel() * t.element_size() for t in c if isinstance(t, torch.Tensor) and t.shape[0] == 9) for c in (big, small)]
    assert sizes[1] * 3 < sizes[0]
    with pytest.raises(ValueError):
        model("wide", "bfloat16", "fp4").new_cache(2, 9, 16)
    name = next(iter(hm.CONFIGS))
    with pytest.raises(TypeError):
        fedatar.load(hm.CONFIGS[name], hm.weights(hm.CONFIGS[name]), "cuda", cache="fp4")
    cfg = dict(vm.CONFIGS["one"], layers=vm.CONFIGS["one"]["layers"][:1], loop=None)
    with pytest.raises(ValueError):
        veredra.load(cfg, vm.weights(cfg), "cuda", cache="fp4")
    with pytest.raises(ValueError):
        veredra.load(vm.CONFIGS["one"], vm.weights(vm.CONFIGS["one"]), "cuda", cache="int3")


@pytest.mark.parametrize("cache", (None, "fp4"))
def test_a_graph_that_takes_pages_gives_the_tokens_of_a_plain_session(cache):
    """Prompts, then decoding captured once: pages are taken inside the graph, over many page borders, and given back."""
    from bitexact_llm_b200.decode import GraphDecoder, Session
    eng = model("looped", "bfloat16", cache)
    prompts = [np.random.RandomState(s).randint(0, 130, n).tolist() for s, n in enumerate((70, 3, 64, 1))]

    def start(**kw):
        ses = Session(eng, 4, 320, **kw)
        h = torch.stack([x[-1] for x in ses.feed(list(enumerate(prompts)))])
        rows = torch.zeros(4, 4, dtype=torch.long, device="cuda")
        rows[:, 0] = torch.arange(4)
        rows[:, 2], rows[:, 3] = 7, 10
        return ses, h, rows

    from bitexact_llm_b200.vllm_plugin import sampler
    ses, h, rows = start()
    want = []
    for t in range(140):
        y = sampler.sample_rows(eng.logits(h), rows, eng.ln, eng.FR)
        want.append(y.tolist())
        rows[:, 1] += 1
        h = ses.step(y)
    ses, h, rows = start(pages=20, perm_seed=3, on_device=True)
    g = GraphDecoder(ses, rows, h, warmup=0)
    assert [g.step().tolist() for _ in range(140)] == want
    assert ses.lens.tolist() == [70 + 140, 3 + 140, 64 + 140, 1 + 140]
    ses.check()
    used = sum(-(-n // 64) for n in ses.lens.tolist())
    assert int(ses.pool.top) == 20 - used
    for s in range(4):
        ses.release(s)
    assert int(ses.pool.top) == 20 and sorted(ses.pool.free.tolist()) == list(range(1, 21)) and not ses.lens.any()


def test_a_full_pool_and_long_sequences_are_told():
    from bitexact_llm_b200.decode import Session
    eng = model("one", "bfloat16", "fp4")
    ses = Session(eng, 3, 128, pages=2, on_device=True)
    ses.feed([(0, [1] * 64), (1, [2] * 64)])
    with pytest.raises(MemoryError):
        ses.feed([(2, [1])])
    keep = ses.lens.clone()
    ses.step(torch.tensor([1, 1, 1]).cuda())
    with pytest.raises(MemoryError):
        ses.check()
    assert torch.equal(ses.lens, keep)
    ses.release(1)
    ses.feed([(0, [3] * 64)])
    with pytest.raises(ValueError):
        ses.feed([(0, [3])])
    with pytest.raises(ValueError):
        ses.step(torch.tensor([1, 1, 1]).cuda(), pos=ses.lens)
    with pytest.raises(ValueError):
        Session(eng, 3, 128, on_device=True)
    with pytest.raises(ValueError):
        Session(eng, 3, 128).step(torch.tensor([1, 1, 1]).cuda(), active=torch.ones(3, dtype=torch.bool).cuda())


def test_prefill_from_a_pool_on_the_device():
    from bitexact_llm_b200.decode import Session
    eng = model("looped", "bfloat16", "fp4")
    prompts = torch.tensor(np.random.RandomState(5).randint(0, 130, (3, 80)))
    lens = torch.tensor([80, 17, 64])
    a, b = Session(eng, 3, 160), Session(eng, 3, 160, pages=9, on_device=True)
    assert torch.equal(a.prefill(prompts, lens, chunk_rows=60), b.prefill(prompts, lens, chunk_rows=60))
    y = torch.tensor([1, 2, 3]).cuda()
    assert torch.equal(a.step(y), b.step(y)) and a.lens.tolist() == b.lens.tolist() == [81, 18, 65]
    b.check()


def test_an_integer_engine_from_a_pool_on_the_device():
    from bitexact_llm_b200.decode import Session
    from bitexact_llm_b200.exact import consts
    from bitexact_llm_b200.vllm_plugin.exact_run import ExactEngine
    cfg = dict(consts.LLAMA_1B, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
               head_dim=64, vocab_size=500)
    eng = ExactEngine(consts.build(cfg, consts.random_state_dict(cfg, seed=1, device="cuda"), n_pos=256), "cuda")
    a, b = Session(eng, 2, 128), Session(eng, 2, 128, pages=16, on_device=True)
    for ses in (a, b):
        ses.feed([(0, list(range(30))), (1, [5])])
    for t in range(20):
        y = torch.tensor([t, 3 * t]).cuda()
        assert torch.equal(a.step(y), b.step(y))
    b.check()


def test_generate_and_score_with_log_probabilities():
    from bitexact_llm_b200.decode import Session, generate, score
    eng = model("looped", "bfloat16", "fp4")
    prompts = [np.random.RandomState(s).randint(0, 130, n).tolist() for s, n in enumerate((20, 1, 7))]
    ids = torch.zeros(3, 20, dtype=torch.long)
    for i, p in enumerate(prompts):
        ids[i, :len(p)] = torch.tensor(p)
    lens = torch.tensor([20, 1, 7])
    plain, _ = generate(eng, ids, 6, 1, 1, lens=lens, hashes=False)
    toks, _, p = generate(eng, ids, 6, 1, 1, lens=lens, hashes=False, logprobs=4)
    assert torch.equal(toks, plain) and p.logp.shape == (3, 6) and p.top_ids.shape == (3, 6, 4)
    for r in score(eng, prompts, 3):
        assert r.top_ids.shape[1] == 3 and (r.logp <= 0).all()
    got = score(eng, prompts, 3)
    assert [len(r.logp) for r in got] == [19, 0, 6] and got[1].top_ids.shape == (0, 3)
    x = Session(eng, 3, 32).feed(list(enumerate(prompts)))
    same(got[0], reference(eng.logits(x[0][:-1]).cpu(), torch.tensor(prompts[0][1:]), 3), 130)
    # portions of any size give the same
    again = score(eng, prompts, 3, chunk_rows=4)
    assert all(torch.equal(a, b) for u, v in zip(got, again) for a, b in zip(u, v))
    with pytest.raises(ValueError):
        score(eng, [[1], []])


def test_commands(tmp_path):
    cfg = vm.CONFIGS["one"]
    hm.save_folder(str(tmp_path), cfg, vm.weights(cfg))
    run = lambda *a: subprocess.run([sys.executable, "-m", "bitexact_llm_b200", *a], cwd=ROOT, capture_output=True, text=True)
    r = run("generate", "--model", str(tmp_path), "--prompt", "1,2,3", "--prompt", "4", "--max-new", "5", "--cache", "fp4", "--logprobs", "2")
    assert r.returncode == 0, r.stderr
    lines = [json.loads(l) for l in r.stdout.splitlines()]
    assert len(lines) == 2 and all(len(l["tokens"]) == len(l["logprobs"]) == len(l["top"]) == 5 and l["rank"] == [1] * 5 for l in lines)
    assert all(l["top"][i][0][0] == l["tokens"][i] and abs(l["top"][i][0][1] - l["logprobs"][i]) < 1e-6 for l in lines for i in range(5))
    r = run("score", "--model", str(tmp_path), "--prompt", "1,2,3", "--cache", "fp4", "--top", "1")
    assert r.returncode == 0, r.stderr
    line = json.loads(r.stdout)
    assert line["tokens"] == [2, 3] and len(line["logprobs"]) == 2 and all(math.exp(v) <= 1 for v in line["logprobs"])
    assert run("score", "--model", str(tmp_path), "--prompt", "1,2", "--cache", "int3").returncode != 0
