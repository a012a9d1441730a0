"""Whole models that cache in 4 bits, and the log probabilities of what they read and write, through the session."""
import json
import os
import subprocess
import sys

import pytest
import torch

import citlali_b200 as cb
import plain_cache4
import plain_qwen3 as plain
from citlali_b200 import ops
from citlali_b200.engine.step import pack_step
from citlali_b200.parts.base import part_class
from helpers import random_tokens, tiny_config
from test_gpu_parts import DEV, InterleavedRotary, close, handles, plain_interleaved_rotary, tol

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load(path, dtype, max_context=256, **more):
    return cb.InferenceSession().load_model(path, max_context=max_context, dtype=dtype, max_batch=4, cache_dtype="int4", **more)


# (tokens whose keys and values all have codes that 32-bit arithmetic settles: see below)
@pytest.mark.parametrize("name,length,seed", [("A", 40, 4), ("B", 70, 4), ("C", 20, 3)])
def test_logits_follow_the_plain_model_with_rounded_keys_and_values(model_dirs, monkeypatch, name, length, seed):
    cfg, w = plain.load_folder(model_dirs[(name, "float32")])
    tokens = random_tokens(cfg["vocab_size"], length, seed)
    nearest = [1.0]

    def rounded(x):
        c, b = plain_cache4.quantised(x)
        s = plain_cache4.scale_of_byte(b)[..., None]
        g = x.unflatten(-1, (-1, 16)) / s
        nearest.append(float(((g - torch.floor(g)) - 0.5).abs().min()))
        wanted = x.unflatten(-1, (-1, 16)).abs().amax(-1) / 7
        table = plain_cache4.scale_of_byte(torch.arange(168))
        middles = (table[1:] + table[:-1]) / 2
        nearest.append(7 * float(((wanted[..., None] - middles).abs().amin(-1) / wanted).min()))
        return plain_cache4.values(plain_cache4.pack(c), b)
    before = plain.causal_attention
    monkeypatch.setattr(plain, "causal_attention", lambda q, k, v, nq, nkv, window=None: before(q, rounded(k), rounded(v), nq, nkv, window))
    want = plain.model_logits(cfg, w, tokens)
    # A code is settled where the element is further from the middle between two than 32-bit arithmetic can move it: keys and values
    # are within 2^-18 of their size here, 7 codes' worth of that in steps.
    assert min(nearest) > 7 * 2.0 ** -18
    session = load(model_dirs[(name, "float32")], "float32")
    slot = session.acquire()
    got = session.step([cb.StepEntry(slot, tokens, range(length))]).cpu().double()
    assert float((got - want).abs().max()) <= 2e-5 * float(want.abs().max())         # the 32-bit path's own bound


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_cache_holds_nine_thirty_seconds_of_bfloat16(model_dirs, dtype):
    packed, wide = load(model_dirs[("D", "bfloat16")], dtype), cb.InferenceSession().load_model(
        model_dirs[("D", "bfloat16")], max_context=256, dtype="bfloat16", max_batch=4)
    assert packed.cache.bytes() * 32 == wide.cache.bytes() * 9


def test_in_32_bits_it_does_not_matter_how_tokens_are_cut_into_steps(model_dirs):
    session = load(model_dirs[("B", "float32")], "float32")
    tokens = random_tokens(1000, 90, 5)
    other = random_tokens(1000, 33, 6)
    a, b, c = session.acquire(), session.acquire(), session.acquire()
    whole = session.step([cb.StepEntry(a, tokens, range(90))])
    cut = [session.step([cb.StepEntry(b, tokens[:41], range(41)), cb.StepEntry(c, other, [32])])[:41]]
    cut.append(session.step([cb.StepEntry(b, tokens[41:64], range(23))]))
    for t in tokens[64:]:
        cut.append(session.step([cb.StepEntry(b, [t], [0])]))
    assert torch.equal(whole, torch.cat(cut))


def test_captured_decoding_gives_the_bits_of_plain_steps(model_dirs):
    prompts = [random_tokens(1536, n, n) for n in (5, 130, 64)]
    made = []
    for graphs in (True, False):
        session = cb.InferenceSession()
        session.use_graphs = graphs
        session.load_model(model_dirs[("D", "bfloat16")], max_context=512, max_batch=3, cache_dtype="int4")
        assert (session.runner is not None) == graphs
        for _ in range(2):                               # the second time over pages that hold the first's keys
            made.append([r.tokens for r in session.generate(prompts, cb.GenerationOptions(max_new_tokens=20, max_context=512, stop_ids=[]))])
    assert all(m == made[0] for m in made[1:])


def test_decoding_and_prompts_agree_in_bfloat16(model_dirs):
    """Token by token, in runs or as one prompt: the same cache, so the same logits up to the paths' own roundings (2.5e-2 of the row's
    largest, as the replays of a cache of 16 bits hold it) wherever bfloat16 keys come out alike."""
    session = load(model_dirs[("D", "bfloat16")], "bfloat16", max_context=512)
    tokens = random_tokens(1536, 100, 9)
    a, b = session.acquire(), session.acquire()
    whole = session.step([cb.StepEntry(a, tokens, range(100))])
    parts = [session.step([cb.StepEntry(b, tokens[:50], range(50))]), session.step([cb.StepEntry(b, tokens[50:70], range(20))])]
    for t in tokens[70:]:
        parts.append(session.step([cb.StepEntry(b, [t], [0])]))
    parts = torch.cat(parts)
    off = (whole - parts).norm(dim=1) / whole.norm(dim=1)
    # a layer's rows differ by bfloat16 roundings (2^-9 of a row's norm or less), a code that flips by it moves one element a step of
    # at most 2/7 of the group's largest: a share of the elements of about 7 2^-8 does, so about sqrt(7 / 2^8) 2 / 7 = 5 % of a key's norm
    assert float(off.max()) < 0.10, off


@pytest.mark.parametrize("dtype,cache_dtype", [("float32", "int4"), ("bfloat16", "int4"), ("bfloat16", None)])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_generation_says_what_scoring_says(model_dirs, dtype, cache_dtype, temperature):
    stored = "float32" if dtype == "float32" else "bfloat16"
    session = cb.InferenceSession().load_model(model_dirs[("B", stored)], max_context=256, dtype=dtype, max_batch=3, cache_dtype=cache_dtype)
    prompts = [random_tokens(1000, n, n) for n in (3, 50, 17, 1)]
    options = cb.GenerationOptions(max_new_tokens=9, max_context=256, temperature=temperature, seed=4, stop_ids=[], logprobs=4)
    results = session.generate(prompts, options)
    plainly = session.generate(prompts, cb.GenerationOptions(max_new_tokens=9, max_context=256, temperature=temperature, seed=4, stop_ids=[]))
    assert [r.tokens for r in results] == [r.tokens for r in plainly] and plainly[0].logprobs is None
    for r in results:
        assert len(r.logprobs) == len(r.entropies) == len(r.alternatives) == 9 and all(len(a) == 4 for a in r.alternatives)
        for token, lp, beside in zip(r.tokens, r.logprobs, r.alternatives):
            assert [v for _, v in beside] == sorted((v for _, v in beside), reverse=True)
            if temperature == 0.0:
                assert beside[0] == (token, lp)
            assert all(lp <= v or token in [i for i, _ in beside] for _, v in beside[:1])
    session.SCORE_ROWS = 23                              # in portions, several texts at a time
    texts = [p + r.tokens for p, r in zip(prompts, results)]
    scored = session.score(texts, top=4)
    for p, r, s in zip(prompts, results, scored):
        assert len(s.logprobs) == len(s.entropies) == len(s.alternatives) == len(p) + 8
        if dtype == "float32":                           # the same logits bit by bit, so the same numbers
            assert s.logprobs[len(p) - 1:] == r.logprobs and s.entropies[len(p) - 1:] == r.entropies
            assert s.alternatives[len(p) - 1:] == r.alternatives
    assert session.cache.slots.free_count == 3
    assert session.details is None


def test_a_generation_within_a_generation(model_dirs):
    session = cb.InferenceSession().load_model(model_dirs[("A", "float32")], max_context=64, dtype="float32", max_batch=2)
    options = cb.GenerationOptions(max_new_tokens=4, max_context=64, stop_ids=[], logprobs=2)
    prompt = random_tokens(512, 5, 1)
    [alone] = session.generate([prompt], options)

    def another(request, token):
        session.generate([[3, 1]], cb.GenerationOptions(max_new_tokens=1, max_context=64, stop_ids=[]))
        session.score([[3, 1, 2]])
    [within] = session.generate([prompt], options, on_token=another)
    assert (within.tokens, within.logprobs, within.alternatives) == (alone.tokens, alone.logprobs, alone.alternatives)
    assert len(alone.logprobs) == 4 and session.details is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [48, 64])
@pytest.mark.parametrize("variant", ["plain", "window", "no_norm_no_rotation", "position_with_apply", "reader"])
def test_a_layer_whatever_its_position_encoding(dtype, d, variant):
    """The layer alone: what it caches lies within its groups' steps of the plain keys and values, and its rows are the plain
    attention's over what it cached.  ``reader``: a second layer without keys reads the first one's."""
    params = {"hidden_size": 40, "num_heads": 6, "num_kv_heads": 2, "head_dim": d, "qk_norm_eps": 1e-5, "window": None,
              "position": {"kind": "rotary_half_split", "theta": 3e4, "rotary_dim": d}}
    norms, rotate = True, True
    if variant == "window":
        params["window"] = 9
    if variant == "no_norm_no_rotation":
        params.update(qk_norm_eps=None, position={"kind": "none"})
        norms = rotate = False
    if variant == "position_with_apply":
        cb.register_part("position", "interleaved_rotary", InterleavedRotary, replace=True)
        params["position"] = {"kind": "interleaved_rotary", "theta": 3e4}
        rotate = "interleaved"
    ctx = cb.BuildContext(DEV, dtype, torch.zeros(4, dtype=torch.int32, device=DEV), packed4=True)
    attn = part_class("mixer", "gqa_attention")(params, "a")
    h, w = handles(attn, dtype, gain_spread=0.5)
    attn.bind(h, ctx)
    parts = [attn]
    if variant == "reader":
        parts.append(part_class("mixer", "gqa_attention")(dict(params, kv_projection=False), "a"))
        parts[1].bind(h, ctx)
    cache = cb.SequenceCache([attn.cache_requirement()], 2, 64 * 6, 64 * 3, dtype, DEV)
    T, nq, nkv = 75, 6, 2
    x = torch.randn(T, 40, generator=torch.Generator().manual_seed(d)).to(dtype)
    project = lambda name, n: plain.linear(x.double(), w[f"a.{name}_proj.weight"]).view(T, n, d)
    q, k, v = project("q", nq), project("k", nkv), project("v", nkv)
    if norms:
        q, k = (plain.head_rms_norm(y, w[f"a.{n}_norm.weight"], 1e-5) for y, n in ((q, "q"), (k, "k")))
    if rotate:
        turn = plain_interleaved_rotary if rotate == "interleaved" else plain.rotary_half_split
        q, k = (turn(y, list(range(T)), 3e4) for y in (q, k))
    other = cache.acquire()
    for pieces in ([(0, T)], [(0, 40)] + [(t, t + 1) for t in range(40, T)]):
        slot, made, held = cache.acquire(), [[] for _ in parts], []
        for lo, hi in pieces:
            batch = pack_step([cb.StepEntry(slot, [0] * (hi - lo), [])], [cache.length(slot)], 10, DEV)
            cache.reserve(slot, hi)
            for part, rows in zip(parts, made):
                rows.append(part.forward(x[lo:hi].to(DEV).contiguous(), batch, cache.view(0), torch.zeros(hi - lo, 40, device=DEV)))
            held.append([y.cpu().double() for y in ops.cache4_read(cache.view(0), batch.row_slot, batch.row_pos, dtype=torch.float32)])
            cache.commit(slot, hi)
        cache.release(slot)
        keys, values = (torch.cat(y) for y in zip(*held))
        for have, want in ((keys, k), (values, v)):
            # half a step, at most (1 + 2^-4) most / 14, or what a scale rounded down cuts off the largest, 2^-4 of it: below 0.08 most;
            # and the paths' own roundings, as for the other layers' tests
            most = want.unflatten(-1, (-1, 16)).abs().amax(-1, keepdim=True).expand(T, nkv, d // 16, 16).flatten(-2)
            assert ((have - want).abs() <= 0.08 * most + tol(dtype) * float(want.abs().max())).all()
        rows = plain.causal_attention(q, keys, values, nq, nkv, window=params["window"]).reshape(T, nq * d)
        want = plain.linear(rows, w["a.o_proj.weight"])
        for part_rows in made:
            close(torch.cat(part_rows), want, dtype)
    cache.release(other)


def test_scoring_follows_the_plain_model(model_dirs):
    cfg, w = plain.load_folder(model_dirs[("A", "float32")])
    session = cb.InferenceSession().load_model(model_dirs[("A", "float32")], max_context=128, dtype="float32", max_batch=2)
    texts = [random_tokens(512, 30, 1), [7], random_tokens(512, 2, 2)]
    found = session.score(texts)
    assert found[1].logprobs == [] and found[1].entropies == [] and all(len(a) == 0 for a in found[0].alternatives)
    for text, f in zip(texts, found):
        if len(text) < 2:
            continue
        logits = plain.model_logits(cfg, w, text)
        lp = torch.log_softmax(logits, -1)
        want = lp[torch.arange(len(text) - 1), torch.tensor(text[1:])]
        bound = 4e-5 * float(logits.abs().max()) + 1e-5  # the logits' own bound twice (an entry's and the sum's), and the kernel's
        assert float((torch.tensor(f.logprobs, dtype=torch.float64) - want).abs().max()) <= bound
        entropy = -(lp.exp() * lp).sum(-1)[:-1]
        assert float((torch.tensor(f.entropies, dtype=torch.float64) - entropy).abs().max()) <= 8 * bound        # (entropies here are below 7)


def test_refusals(model_dirs):
    session = load(model_dirs[("A", "float32")], "float32", max_context=32)
    for bad, words in [(lambda: session.score([[1, 2], []]), "no tokens"), (lambda: session.score([[1, 600]]), "out of vocab"),
                       (lambda: session.score([[600, 1]]), "out of vocab"), (lambda: session.score([[1] * 34]), "context"),
                       (lambda: session.score([[1, 2]], top=33), "0 to 32"),
                       (lambda: session.generate([[1]], cb.GenerationOptions(logprobs=40)), "logprobs")]:
        with pytest.raises(cb.CitlaliError, match=words):
            bad()
    assert session.cache.slots.free_count == 4
    assert len(session.score([[1] * 33])[0].logprobs) == 32           # the last token need not be read
    with pytest.raises(cb.CitlaliError, match="cache_dtype"):
        cb.InferenceSession().load_model(model_dirs[("A", "float32")], dtype="float32", cache_dtype="int3")


def test_command_line(model_dirs):
    out = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "citlali_cli"), "--model", model_dirs[("D", "bfloat16")], "--prompt-ids", "1,2,3",
                          "--prompt-ids", "4,5", "--max-new-tokens", "4", "--cache-dtype", "int4", "--logprobs", "2", "--json"],
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr
    results = json.loads(out.stdout)["results"]
    assert all(len(r["logprobs"]) == len(r["tokens"]) and all(len(a) == 2 for a in r["alternatives"]) for r in results)
