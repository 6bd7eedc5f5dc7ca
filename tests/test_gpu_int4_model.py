"""Models with weights and cache in 4 bits, through the engine and the command line."""
import contextlib
import io

import pytest
import torch

import tiny

pytestmark = pytest.mark.gpu
PAGE = {"C": 16, "D": 64, "E": 64, "G": 16}
LENGTHS = {"C": [90, 41, 7], "D": [300, 33, 129], "E": [260, 70, 1]}
HELD = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


def load(folder, **more):
    from garlic_inference_b200 import AutoModel
    return AutoModel.from_pretrained(folder, device=0, **more)


@pytest.mark.parametrize("name", ["C", "D", "E"])
def test_weights_in_4_bits_compute_what_the_codes_stand_for(name, model_dirs, tmp_path):
    """Against the plain implementation with the numbers that the codes stand for as float32 weights: the bfloat16 engine's own
    bound, whole prompts, token by token and in batches."""
    import shutil
    from garlic_inference_b200.ops import int4
    from garlic_inference_b200.weights import Checkpoint
    from garlic_inference_b200.weights.safetensors_io import write_safetensors
    folder = model_dirs(name)
    ckpt = Checkpoint(folder)
    tensors = {}
    for n in ckpt.names():
        t = ckpt.tensor(n).clone()
        if any(f"{p}.weight" in n for p in HELD):
            t = int4.dequantize_weight(int4.quantize_weight(t.cuda()), torch.float32).cpu()
        tensors[n] = t
    shutil.copy(folder / "config.json", tmp_path / "config.json")
    write_safetensors(tmp_path / "model.safetensors", tensors)
    reqs = tiny.random_requests(tiny.TINY[name]["cfg"]["vocab_size"], LENGTHS[name], seed=5)
    want = tiny.plain_logits(tmp_path, reqs)
    max_tokens = sum(-(-n // 64) * 64 for n in LENGTHS[name])
    model = load(folder, max_tokens=max_tokens, page_size=PAGE[name], weights="int4")
    plain = load(folder, max_tokens=64)
    assert model.model.weight_bytes() < plain.model.weight_bytes()
    for what, trace in (("whole", tiny.trace_whole(reqs)), ("one by one", tiny.trace_tail_by_one(reqs, tail=20)),
                        ("batched", tiny.trace_batched(reqs, [["r0", "r1", "r2"]], prompt_frac=0.5))):
        got = tiny.run_trace_in_process(model, trace)
        tiny.assert_covers(got, reqs)
        tiny.compare(got, want, tiny.TOL["bfloat16"], f"{name} {what}")


@pytest.mark.parametrize("name,page", [("D", 64), ("E", 16), ("E", 64), ("G", 7)])
def test_attention_over_a_cache_in_4_bits_is_its_operators_in_turn(name, page, model_dirs, monkeypatch):
    """What the layers hand to the operators: prompts of many and of few tokens, single tokens, a window whose pages are
    given back.  Every call's result is held against the formulas in 64 bits over the pages as they are."""
    import plain_int4 as plain
    from garlic_inference_b200.ops import int4
    model = load(model_dirs(name), max_tokens=1024, page_size=page, cache="int4", use_graphs=False)
    seen = {"decode": 0, "prompt": 0}
    decode, prompt = int4.attention_decode, int4.attention_prompt

    def check(got, q, k, v, table, spans, scale, window, wide):
        filled = table.clamp(min=0)                          # pages given back lie behind the window
        want, bound = plain.attention(q, k, v, filled, spans, scale, window)
        if wide:                                             # keys and values rounded to bfloat16 on the way, probabilities too
            for s, r, n, p in spans:
                kc, ks, kl = plain.sequence(k, filled[s], p + n)
                vc, vs, vl = plain.sequence(v, filled[s], p + n)
                kk, vv = plain.values(kc, ks, kl, 64), plain.values(vc, vs, vl, 64)
                heads, d = q.shape[1:]
                for h in range(heads):
                    e = h // (heads // k.shape[1])
                    off = 2 ** -8 * (q[r:r + n, h].double().abs() @ kk[e].abs().t()).amax(1, keepdim=True) * scale
                    bound[r:r + n, h * d:(h + 1) * d] += (2 * off + 2 ** -7) * vv[e].abs().amax(0)[None]
        assert bool(((got.double() - want).abs() <= bound + 1e-30).all())

    def on_decode(q, k, v, table, pos, slot, scale, window, status, **kw):
        got = decode(q, k, v, table, pos, slot, scale, window, status, **kw)
        spans = [(s, i, 1, p) for i, (s, p) in enumerate(zip(slot.tolist(), pos.tolist()))]
        check(got, q, k, v, table, spans, scale, window, False)
        seen["decode"] += 1
        return got

    def on_prompt(q, k, v, table, runs, blocks, scale, window, status):
        got = prompt(q, k, v, table, runs, blocks, scale, window, status)
        check(got, q, k, v, table, [(r[0], r[1], r[2], r[3]) for r in runs.tolist()], scale, window, True)
        seen["prompt"] += 1
        return got

    monkeypatch.setattr(int4, "attention_decode", on_decode)
    monkeypatch.setattr(int4, "attention_prompt", on_prompt)
    vocab = tiny.TINY[name]["cfg"]["vocab_size"]
    reqs = tiny.random_requests(vocab, [230, 33, 129], seed=3)
    a, b, c = (model.alloc_slot() for _ in range(3))
    r = [reqs[f"r{i}"] for i in range(3)]
    model.step([(a, r[0][:200], [199]), (b, r[1][:30], [29])])
    model.step([(a, r[0][200:203], [2]), (b, r[1][30:32], [1]), (c, r[2][:5], [4])])
    model.step([(c, r[2][5:128], [122]), (a, r[0][203:204], [0])])
    for i in range(3):
        out = model.step([(a, [r[0][204 + i]], [0]), (c, [r[2][128 - i]], [0]), (b, [r[1][i]], [0])])
        assert bool(torch.isfinite(out).all())
    model.engine.check()
    layers = tiny.TINY[name]["cfg"]["num_hidden_layers"]
    assert seen == {"decode": 3 * layers, "prompt": 3 * layers}


@pytest.mark.parametrize("weights,cache", [("int4", None), (None, "int4"), ("int4", "int4")])
@pytest.mark.parametrize("name", ["D", "E"])
def test_recorded_steps_give_the_bits_of_eager_ones(name, weights, cache, model_dirs):
    """Batches of 1, 2 and 4, which fill their recorded step, so that both run the same kernels at the same sizes."""
    vocab = tiny.TINY[name]["cfg"]["vocab_size"]
    reqs = tiny.random_requests(vocab, [70, 130, 20, 64], seed=8)
    models = [load(model_dirs(name), max_tokens=2048, weights=weights, cache=cache, use_graphs=g) for g in (True, False)]
    out = []
    for m in models:
        got = []
        for n in (1, 2, 4):
            slots = [m.alloc_slot() for _ in range(n)]
            got.append(m.step([(s, reqs[f"r{i}"][:-6], [0]) for i, s in enumerate(slots)]))
            for t in range(6):
                got.append(m.step([(s, [reqs[f"r{i}"][t - 6]], [0]) for i, s in enumerate(slots)]).clone())
            for s in slots:
                m.free_slot(s)
        m.engine.check()
        out.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*out))
    bits = models[0].engine.cache.bytes_per_token()
    assert (bits < load(model_dirs(name), max_tokens=64).engine.cache.bytes_per_token() / 3) == (cache is not None)


def test_generation_is_repeatable_and_gives_its_pages_back(model_dirs):
    model = load(model_dirs("E"), max_tokens=768, weights="int4", cache="int4")
    prompts = list(tiny.random_requests(400, [150, 3, 64, 65, 200, 10], seed=1).values())
    first = model.generate(prompts, max_new_tokens=40, max_batch=3)
    assert first == model.generate(prompts, max_new_tokens=40, max_batch=3) and all(len(o) == 40 for o in first)
    cache = model.engine.cache
    assert cache.slots.n_free == cache.max_slots and all(g.host.pool.n_free == g.host.pool.n_pages for g in cache.groups)


@pytest.mark.parametrize("module,name", [("tiny_fivitar", "mix"), ("tiny_kenovik", None), ("tiny_dugopel", None), ("tiny_zogulorn", None),
                                         ("tiny_nezolorn", None), ("tiny_netolorn", None)])
def test_other_architectures_pack_their_feed_forwards_or_say_that_they_pack_nothing(module, name, tmp_path):
    """Every model either runs with what it packs, graphs included, or refuses; none has keys and values for 4 bits."""
    import importlib
    tiny_of = importlib.import_module(module)
    ran = 0
    for n in [name] if name else list(tiny_of.TINY):
        folder = tmp_path / n
        folder.mkdir()
        folder = tiny_of.write_model(n, folder)
        try:
            model = load(folder, max_tokens=256, weights="int4")
        except ValueError as e:
            assert "none of this model's parts" in str(e)
            continue
        out = model.generate([[1, 2, 3, 4, 5], [7, 8]], max_new_tokens=6)
        assert [len(o) for o in out] == [6, 6] and out == model.generate([[1, 2, 3, 4, 5], [7, 8]], max_new_tokens=6)
        ran += 1
        with pytest.raises(ValueError, match="none of this model's mixers"):
            load(folder, max_tokens=256, cache="int4")
    assert ran


def test_float32_activations_take_weights_in_4_bits_and_no_such_cache(model_dirs):
    model = load(model_dirs("D"), max_tokens=256, dtype="float32", weights="int4")
    assert len(model.generate([[1, 2, 3]], max_new_tokens=5)[0]) == 5
    with pytest.raises(ValueError, match="4 bits"):
        load(model_dirs("D"), max_tokens=256, dtype="float32", cache="int4")
    with pytest.raises(ValueError, match="4 bits"):
        load(model_dirs("A"), max_tokens=256, cache="int4")              # heads of 16


def test_the_command_line(model_dirs):
    from garlic_inference_b200.cli import main
    outs = []
    for more in ([], ["--weights", "int4", "--cache", "int4"]):
        text = io.StringIO()
        with contextlib.redirect_stdout(text):
            assert main([str(model_dirs("D")), "--prompt-ids", "1,2,3", "--max-new-tokens", "4", "--print-logits", "3", *more]) == 0
        outs.append(text.getvalue())
    assert all("Tok/s:" in o and "Logits 0:" in o for o in outs) and outs[0] != outs[1]
