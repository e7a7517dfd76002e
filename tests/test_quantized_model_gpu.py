"""Llama with quantised layers through the engine (prompts whole, in unequal batches, the last tokens one by one with captured
decode steps) and through the entry points, against the plain restatements.

Tolerances.  4-bit weights: that of bfloat16 models, 2% of the largest logit.  8-bit rows: the oracle rounds where the engine does, but
what it rounds differs from the engine's by up to a step of bfloat16, 2^-8 of a value.  e4m3 values lie at least 2^-4 apart, so at
most one value in 2^4 comes out on the other side of a border, and then by at most 2^-3 of itself: a row's difference is at
most sqrt(2^-4) 2^-3 = 2^-5 of it, in the root mean square, and so is that of a product with independent weights; two products
follow one another in a sublayer, sqrt(2) 2^-5, and the stream, a sum of independent sublayers, is no further off.  The largest
of up to 10^5 differences is below 4.5 of their root mean square, the largest of 256 logits and more above 3.1 of theirs:
sqrt(2) 2^-5 4.5 / 3.1 = 0.064 of the largest logit."""
import os
import subprocess
import sys

import pytest
import torch

import plain_quantized as pq
from tiny_models import TINY, tiny_prompts

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KINDS = [("fp8", None), ("int4", 32), ("int4", 128)]


def config(kind, group):
    return {"linear_type": kind} if group is None else {"linear_type": kind, "group_size": group}


@pytest.fixture(scope="module")
def built(tiny_folders):
    from fms_b200.models import get_model

    cache = {}

    def get(which, kind, group):
        key = which, kind, group
        if key not in cache:
            folder = tiny_folders[which]
            model = get_model("hf_pretrained", model_path=folder, device_type="cuda", data_type="bf16", linear_config=config(kind, group))
            cache[key] = model, pq.Fp8Llama(folder) if kind == "fp8" else pq.Int4Llama(folder, group)
        return cache[key]

    return get


def close(got, want, kind):
    torch.testing.assert_close(got.double().cpu(), want, atol=(0.064 if kind == "fp8" else 0.02) * want.abs().max().item(), rtol=0.02)


def requests(which):
    g = torch.Generator().manual_seed(7)
    cfg = TINY[which][0]
    lengths = [1, 5, 33, 64] + ([90] if cfg["max_position_embeddings"] >= 128 else []) + ([300] if cfg["max_position_embeddings"] >= 512 else [])
    return [torch.randint(0, cfg["vocab_size"], (n,), generator=g).tolist() for n in lengths]


@pytest.mark.parametrize("kind,group", KINDS)
@pytest.mark.parametrize("which", ["a", "b", "c", "e"])
def test_prompts_alone_and_the_last_tokens_one_by_one(built, which, kind, group):
    model, oracle = built(which, kind, group)
    engine = model.new_engine(max_tokens=1024)
    for req in tiny_prompts(which) + requests(which):
        want = oracle.logits(req)
        (slot,) = engine.begin(1)
        close(engine.step([slot], [req], [list(range(len(req)))]), want, kind)
        engine.release([slot])
        first = max(1, len(req) - 6)
        if first < len(req):
            (slot,) = engine.begin(1)
            engine.step([slot], [req[:first]], [[]])
            got = torch.cat([engine.step([slot], [[t]], [[0]]) for t in req[first:]])
            engine.release([slot])
            close(got, want[first:], kind)
    engine.check()


@pytest.mark.parametrize("kind,group", KINDS)
@pytest.mark.parametrize("which", ["a", "c"])
def test_unequal_batches(built, which, kind, group):
    model, oracle = built(which, kind, group)
    reqs = requests(which)
    engine = model.new_engine(max_tokens=2048, max_slots=8)
    for batch in (reqs, reqs[::-1][:3]):
        slots = engine.begin(len(batch))
        got = engine.step(slots, batch, [list(range(len(r))) for r in batch])
        close(got, torch.cat([oracle.logits(r) for r in batch]), kind)
        engine.release(slots)
    engine.check()


@pytest.mark.parametrize("kind,group", KINDS)
def test_generation_and_what_a_model_keeps(built, kind, group):
    from fms_b200.utils.generation import generate

    model, oracle = built("a", kind, group)
    prompts = [torch.tensor(p) for p in tiny_prompts("a")[:2]]
    out = generate(model, prompts, max_new_tokens=5, do_sample=False)
    again = generate(model, prompts, max_new_tokens=5, do_sample=False)
    assert [o.tolist() for o in out] == [o.tolist() for o in again]
    steps = []
    generate(model, prompts, max_new_tokens=5, do_sample=False, post_iteration_hook=lambda it, lg, toks, reqs: steps.append(lg.float().cpu()))
    for i, (o, p) in enumerate(zip(out, prompts)):
        close(torch.stack([lg[i] for lg in steps]), oracle.logits(o.tolist()[:-1])[len(p) - 1:], kind)
    state = model.state_dict()
    assert all(isinstance(t, torch.Tensor) for t in state.values())
    kept = [n for n in state if "attn.dense.weight" in n]
    assert kept and all(n.endswith((".values", ".scales") if kind == "fp8" else ".blocks") for n in kept)
    assert state["base_model.embedding.weight"].dtype == torch.bfloat16


def test_layers_as_stored_are_what_they_were(tiny_folders):
    from fms_b200.models import get_model

    req = [5, 17, 3, 200, 9]
    plain = get_model("hf_pretrained", model_path=tiny_folders["a"], device_type="cuda", data_type="bf16")
    named = get_model("hf_pretrained", model_path=tiny_folders["a"], device_type="cuda", data_type="bf16", linear_config={"linear_type": "torch_linear"})
    assert torch.equal(plain(torch.tensor(req)), named(torch.tensor(req)))


def test_the_command_line(tiny_folders):
    for kind in ("fp8", "int4"):
        run = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "fms_inference"), "--model_path", tiny_folders["a"], "--default_dtype", "bf16",
                              "--linear_type", kind, "--linear_group_size", "32", "--prompt_ids", "5,17,3", "--max_new_tokens", "4"],
                             capture_output=True, text=True, timeout=300)
        assert run.returncode == 0, run.stderr[-2000:]
        assert len(run.stdout.strip().split(",")) == 7
