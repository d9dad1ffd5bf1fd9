"""Models whose layers hold their matrices in 8 bits, against the plain decoder with the same roundings.

Tolerance.  Engine and plain decoder round the same numbers to 8 bits, but where the engine's differ in their last bits a number
next to the middle of two steps falls to the other side, and from there on the two see other numbers, whose further roundings
differ as those of any two numbers do: by up to a step, 1/127 of a row's largest value, with a spread of step / sqrt(6).  A row's
largest value is about 3.5 of its rms, so a product's result is off by 3.5 / 127 / sqrt(6) = 1.1 percent of its own size.  Two or
three layers have four such products on the way, each: sqrt(12) of them are 3.9 percent of the stream's rms, and the largest
logit of a row, which the error is related to, is 2.5 to 3 of the rms.  The largest of some thousands of such errors is 3.5 of
their spread: 3.9 * 3.5 / 2.5 = 5.5 percent.  A product without its scales, or with another row's, is off by all of its size."""
import numpy as np
import pytest
import torch

from helpers import CONFIGS, make_folder, random_prompts, scaled_error

pytestmark = pytest.mark.gpu
LENGTHS = {"tiny-llama": [5, 70], "tiny-qwen3": [1, 31, 200], "tiny-odd": [3, 130], "tiny-wide": [40, 330]}
TOLERANCE = {"float32": 0.055, "bfloat16": 0.055 + 0.03}  # with what bfloat16 rounds of its own (helpers.TOL)


@pytest.fixture(scope="module")
def setups(tmp_path_factory):
    from plain import int8
    from plain.files import read_model_folder
    out, root = {}, tmp_path_factory.mktemp("models")
    for name in CONFIGS:
        folder = make_folder(root, name, sharpen=3.0)
        cfg, weights = read_model_folder(folder)
        prompts = random_prompts(cfg["vocab_size"], LENGTHS[name], seed=len(name))
        out[name] = (folder, prompts, [int8.forward_logits(cfg, weights, p) for p in prompts])
    return out


def _engine(folder, dtype, weights="int8"):
    from xeno_rt_b200.engine import Engine, Model
    return Engine(Model.load(folder, dtype=dtype, weights=weights), max_tokens=64 * 24)


def _whole(engine, prompt):
    from xeno_rt_b200.engine import StepEntry
    slot = engine.open_slot()
    logits = engine.step([StepEntry(slot, prompt, list(range(len(prompt))))]).cpu().numpy()
    engine.close_slot(slot)
    return logits


def _one_by_one(engine, prompt, tail):
    from xeno_rt_b200.engine import StepEntry
    slot = engine.open_slot()
    head = len(prompt) - tail
    rows = [engine.step([StepEntry(slot, prompt[:head], list(range(head)))]).cpu().numpy()] if head else []
    rows += [engine.step([StepEntry(slot, [t], [0])]).cpu().numpy() for t in prompt[head:]]
    engine.close_slot(slot)
    return np.concatenate(rows)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_against_the_plain_decoder(setups, name, dtype):
    folder, prompts, wants = setups[name]
    engine = _engine(folder, dtype)
    for prompt, want in zip(prompts, wants):
        assert scaled_error(_whole(engine, prompt), want) < TOLERANCE[dtype]
        tail = min(len(prompt), 12)  # steps of one token, replayed from graphs
        assert scaled_error(_one_by_one(engine, prompt, tail), want) < TOLERANCE[dtype]
    engine.check_errors()


def test_batches_of_unequal_lengths_and_padding_rows(setups):
    from xeno_rt_b200.engine import StepEntry
    folder, prompts, wants = setups["tiny-qwen3"]
    engine = _engine(folder, "bfloat16")
    slots = [engine.open_slot() for _ in prompts]
    heads = [max(1, len(p) - 5) for p in prompts]
    first = engine.step([StepEntry(s, p[:h], [h - 1]) for s, p, h in zip(slots, prompts, heads)], pad_to=sum(heads) + 7).cpu().numpy()
    for row, want, h in zip(first, wants, heads):
        assert scaled_error(row[None], want[h - 1][None]) < TOLERANCE["bfloat16"]
    live = [i for i, (p, h) in enumerate(zip(prompts, heads)) if h < len(p)]
    rows = engine.step([StepEntry(slots[i], [prompts[i][heads[i]]], [0]) for i in live]).cpu().numpy()
    for row, i in zip(rows, live):
        assert scaled_error(row[None], wants[i][heads[i]][None]) < TOLERANCE["bfloat16"]


def test_matrices_take_half_the_bytes_and_the_stored_ones_are_given_up(setups):
    from xeno_rt_b200.engine import Model
    folder = setups["tiny-wide"][0]
    sizes = {}
    for weights in (None, "int8"):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        model = Model.load(folder, dtype="bfloat16", weights=weights)
        torch.cuda.synchronize()
        sizes[weights] = torch.cuda.memory_allocated() - before
        del model
    layers = 2 * (256 * (4 * 128 + 2 * 2 * 128 + 4 * 128) + 3 * 256 * 384)  # elements of the layers' matrices
    assert sizes[None] - sizes["int8"] > 0.9 * layers


def test_command_and_entry_point(setups, capsys):
    from xeno_rt_b200 import GenerateRequest, Runtime
    from xeno_rt_b200.cli import main
    folder, prompts, _ = setups["tiny-wide"]
    request = GenerateRequest(prompts[0], max_tokens=6, temperature=0.0, stop_ids=())
    tokens = Runtime.load(folder, weights="int8").new_session().generate(request)
    assert len(tokens) == 6
    assert main(["generate", "--model", folder, "--prompt-ids", ",".join(map(str, prompts[0])), "--max-tokens", "6",
                 "--temperature", "0", "--repetition-penalty", "1.1", "--weights", "int8", "--stop-ids", ""]) == 0
    assert capsys.readouterr().out.strip() == ",".join(map(str, tokens))


def test_a_random_model_is_the_one_of_its_folder(tmp_path):
    from xeno_rt_b200 import write_random_model
    from xeno_rt_b200.engine import Engine, Model
    raw, seed, _ = CONFIGS["tiny-wide"]
    folder = str(tmp_path / "m")
    write_random_model(folder, raw, seed, "bfloat16")
    prompt = random_prompts(raw["vocab_size"], [20])[0]
    logits = [_whole(Engine(m, max_tokens=256), prompt) for m in (Model.load(folder, weights="int8"),
                                                                  Model.random(raw, seed=seed, weights="int8"))]
    assert np.array_equal(*logits)


def test_layers_that_share_their_tensors(setups):
    """Two layers built from the same tensors, and from copies of them."""
    from xeno_rt_b200.config import load_config
    from xeno_rt_b200.core import parse_dtype
    from xeno_rt_b200.engine import Engine, Model
    from xeno_rt_b200.weights import load_weights
    folder, prompts, _ = setups["tiny-wide"]
    arch, config = load_config(folder)
    logits = []
    for share in (True, False):
        spec = arch.build_spec(config)
        tensors = load_weights(folder, spec.expected_tensors(), parse_dtype("bfloat16"), "cuda:0", spec.ignorable_tensors,
                               fused_groups=spec.fused_groups())
        if share:
            spec.layers[1] = spec.layers[0]
        else:
            for name, (_, part) in spec.layers[0].parts.items():
                for role, source in part.weights.items():
                    tensors[spec.layers[1].parts[name][1].weights[role]].copy_(tensors[source])
        model = Model(spec, tensors, parse_dtype("bfloat16"), "cuda:0", config, weights="int8")
        assert not any(n in tensors for _, part in spec.layers[0].parts.values() if part.kind in ("attention", "swiglu")
                       for n in part.weights.values())
        logits.append(_whole(Engine(model, max_tokens=64 * 24), prompts[0]))
    assert np.array_equal(*logits)
