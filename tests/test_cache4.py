"""The cache in 4 bits and the generation's log probabilities without a device: storage, arguments, refusals, bookkeeping."""
import math

import pytest
import torch

import citlali_b200 as cb
import plain_cache4 as plain
from citlali_b200 import ops
from citlali_b200.cli import parse_args
from citlali_b200.engine.generate import run_generation
from citlali_b200.engine.session import parse_cache_dtype
from helpers import tiny_config
from test_generate_loop import FakeStepper


def test_the_plain_format():
    """The tests' own restatement: every byte's scale, the nearest of them, half-way cases."""
    table = plain.scale_of_byte(torch.arange(168))
    halves = (torch.arange(168, dtype=torch.int16) << 7).view(torch.float16).double() * 8
    assert torch.equal(table, halves) and bool((table[1:] > table[:-1]).all()) and float(table[-1]) == 480.0
    x = torch.zeros(3, 16, dtype=torch.float64)
    x[0, 0] = 7 * (float(table[100]) + float(table[101])) / 2        # between an even byte and an odd one
    x[1, 0] = 7 * (float(table[101]) + float(table[102])) / 2
    x[2, 0] = math.inf
    assert plain.byte_of(x).tolist() == [100, 102, 255]
    c, b = plain.quantised(torch.tensor([[7.0, 0.5, 1.5, -0.5, -1.5, 2.5] + [0.0] * 10]))
    assert b.item() == 15 * 8 - 3 * 8 and c[0, :6].tolist() == [7, 0, 2, 0, -2, 2]        # s = 1
    assert plain.values(plain.pack(c), b)[0, :3].tolist() == [7.0, 0.0, 2.0]


def test_storage():
    reqs = [cb.KVRequirement(2, 32, packed4=True), cb.KVRequirement(2, 32, packed4=True), cb.KVRequirement(2, 32)]
    c = cb.SequenceCache(reqs, 3, 64 * 4, 128, torch.bfloat16, "cpu")
    assert [g.requirement.packed4 for g in c.kv_groups] == [True, False]
    v = c.view(1)
    assert isinstance(v.keys, cb.Packed4) and tuple(v.keys.codes.shape) == (4, 2, 64, 16) and tuple(v.values.scales.shape) == (4, 2, 64, 2)
    assert v.keys.codes.dtype == v.keys.scales.dtype == torch.uint8
    assert v.keys.codes.data_ptr() != c.view(0).keys.codes.data_ptr()
    packed, wide = 2 * 2 * 4 * 2 * 64 * (16 + 2), 2 * 4 * 2 * 64 * 32 * 2
    assert c.bytes() == packed + wide and packed * 32 == 2 * wide * 9
    slot = c.acquire()
    c.reserve(slot, 100)
    c.commit(slot, 100)
    assert c.pages_held() == 4                    # both groups
    c.rewind(slot, 3)
    c.release(slot)
    for bad in (24, 8, 272):
        with pytest.raises(cb.CitlaliError, match="multiples of 16"):
            cb.SequenceCache([cb.KVRequirement(2, bad, packed4=True)], 1, 64, 64, torch.bfloat16, "cpu")


def test_cache_dtype_argument():
    assert parse_cache_dtype("int4", torch.bfloat16) and parse_cache_dtype("int4", torch.float32)
    assert not parse_cache_dtype(None, torch.float32) and not parse_cache_dtype("bf16", torch.bfloat16)
    with pytest.raises(cb.CitlaliError, match="cache_dtype"):
        parse_cache_dtype("int8", torch.bfloat16)
    with pytest.raises(cb.CitlaliError, match="cache_dtype"):
        parse_cache_dtype("float32", torch.bfloat16)


def test_models_whose_mixers_cannot_are_refused():
    ctx = cb.BuildContext(torch.device("cpu"), torch.bfloat16, packed4=True)
    model = cb.DecoderModel(tiny_config("A").to_model_spec(), ctx)
    assert {"cache4", "attention4", "attention4_runs"} <= set(model.kernel_sources())
    from citlali_b200.measure import gidirax_config
    spec = gidirax_config(256, 4, 512).to_model_spec()
    cb.DecoderModel(spec, cb.BuildContext(torch.device("cpu"), torch.bfloat16))
    with pytest.raises(cb.CitlaliError, match="4 bits"):
        cb.DecoderModel(spec, ctx)


def test_tensors_on_the_cpu_are_refused():
    kv = cb.SequenceCache([cb.KVRequirement(1, 16, packed4=True)], 1, 64, 64, torch.float32, "cpu").view(0)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(cb.CitlaliError, match="CUDA"):
        ops.cache4_append(torch.zeros(1, 48), kv, one, one, 1, 1, 16, torch.zeros(8), 16)
    with pytest.raises(cb.CitlaliError, match="CUDA"):
        ops.cache4_read(kv, one, one)
    batch = cb.StepBatch(one, one, one, torch.zeros(2, dtype=torch.int32), one, one, one, slots=[0], past=[0], n_new=[1])
    with pytest.raises(cb.CitlaliError, match="CUDA"):
        ops.cache4_attention(torch.zeros(1, 16), 16, kv, batch, torch.zeros(1, 16), 1, 1, 16, 0, 1.0)
    with pytest.raises(cb.CitlaliError, match="CUDA"):
        ops.token_logprobs(torch.zeros(1, 16), one)
    with pytest.raises(cb.CitlaliError, match="4 bits"):
        ops.cache4_read(cb.KVView(torch.zeros(1, 1, 64, 16), torch.zeros(1, 1, 64, 16), one[None], 64, cb.KVRequirement(1, 16)), one, one)


class TellingStepper(FakeStepper):
    """Says of each token it gives that its log probability is minus its id, its entropy half of it, and names one other."""

    def _tell(self, tokens):
        self.details = cb.TokenDetails([-float(t) for t in tokens], [t / 2 for t in tokens], [[(t + 1, -1.0)] for t in tokens])
        return tokens

    def prefill(self, *a):
        return self._tell(super().prefill(*a))

    def decode(self, *a):
        return self._tell(super().decode(*a))


def test_details_stay_with_their_tokens():
    scripts = {0: [10, 11, 99, 0, 0], 1: [20, 99], 2: [30, 31, 32, 33, 34, 35]}
    options = cb.GenerationOptions(max_new_tokens=4, max_context=64, logprobs=1)
    res = run_generation(TellingStepper(scripts), [[0, 1, 2], [1], [2, 5]], options, [99], 4)
    for r in res:                                   # a stop token is not among the tokens, nor what is said of it
        assert r.logprobs == [-float(t) for t in r.tokens] and r.entropies == [t / 2 for t in r.tokens]
        assert r.alternatives == [[(t + 1, -1.0)] for t in r.tokens]
    assert res[1].tokens == [20]
    none = run_generation(FakeStepper(scripts), [[0, 1, 2]], cb.GenerationOptions(max_new_tokens=2, max_context=64), [99], 4)
    assert none[0].logprobs is None and none[0].alternatives is None
    for bad in (-1, 33):
        with pytest.raises(cb.CitlaliError, match="logprobs"):
            run_generation(FakeStepper(scripts), [[0]], cb.GenerationOptions(max_new_tokens=2, max_context=64, logprobs=bad), [], 4)


def test_details_of_what_the_kernel_gives():
    found = {"logprobs": torch.tensor([-1.0, -2.0]), "entropy": torch.tensor([0.5, 0.25]),
             "top_ids": torch.tensor([[3, 1], [2, -1]], dtype=torch.int32), "top_logprobs": torch.tensor([[-1.0, -3.0], [-2.0, -math.inf]])}
    d = cb.TokenDetails.of(found)
    assert d.logprobs == [-1.0, -2.0] and d.entropies == [0.5, 0.25] and d.alternatives == [[(3, -1.0), (1, -3.0)], [(2, -2.0)]]
    del found["top_ids"], found["top_logprobs"]
    assert cb.TokenDetails.of(found).alternatives == [[], []]


def test_command_line():
    a = parse_args(["citlali_cli", "--model", "m", "--prompt-ids", "1", "--cache-dtype", "int4", "--logprobs", "3"])
    assert a.cache_dtype == "int4" and a.logprobs == 3
    a = parse_args(["citlali_cli", "--model", "m", "--prompt-ids", "1"])
    assert a.cache_dtype is None and a.logprobs is None


def test_which_way_runs_go():
    """By the times that ops._attention4_way works out."""
    def way(past, new, nq=16, nkv=8, d=128, window=0, form=2, tokens=None, codes=True):
        batch = cb.StepBatch(*[torch.zeros(1, dtype=torch.int32)] * 7, slots=list(range(len(new))), past=past, n_new=new)
        return ops._attention4_way(batch, nq, nkv, d, window, lambda: form, 128 // (nq // nkv) if tokens is None else tokens, codes, 148)
    # few columns read the codes, more of them go in tiles that as many blocks share as fit at once, the longest prompts over pages
    assert way([2000], [4]) == ("codes",) and way([2000], [64]) == ("tiles", 0, 8, 8) and way([0], [2048]) == ("tiles", 0, 256, 1)
    assert way([8000] * 4, [6] * 4) == ("codes",) and way([8000] * 4, [16] * 4) == ("tiles", 0, 32, 4) and way([500] * 32, [4] * 32) == ("codes",)
    assert way([5000, 5600, 6300, 7000], [5, 24, 11, 18], 40, window=4096) == ("tiles", 0, 32, 4)
    assert way([300] * 4, [24] * 4, 40) == ("tiles", 0, 32, 1) and way([0], [4096])[0] == "pages"
    assert way([2000, 10, 300], [100, 1, 0])[:2] == ("tiles", 0) and way([0] + [4000] * 63, [512] + [1] * 63)[:3] == ("tiles", 4, 64)
    # sizes that the kernel for tiles does not take
    assert way([2000], [8], tokens=0) == ("codes",) and way([1952], [96], tokens=0) == ("codes",) and way([0], [2048], tokens=0) == ("pages",)
    assert way([2000] * 4, [40] * 4, 40, tokens=0) == ("codes",) and way([1952] * 4, [96] * 4, 40, tokens=0) == ("pages",)
    assert way([100], [64], form=0, tokens=0) == ("codes",) and way([40000], [60], window=128, tokens=0) == ("codes",)
    assert way([0], [100], d=80, form=1, tokens=0, codes=False) == way([0], [20], d=80, form=1, tokens=0, codes=False) == ("pages",) and way([0], [5], d=80, form=1, tokens=0, codes=False) == ("codes",)
