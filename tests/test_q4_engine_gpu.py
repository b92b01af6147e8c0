"""Models whose matrices are held in four bits, through the engine: against the plain implementation on the matrices that the codes stand
for, held to what rounding to bfloat16 costs (`helpers.RoundingJudge`), as the dense engine is."""
import numpy as np
import pytest
import torch

import plain_qwen3 as P
import q4_helpers as q4
from helpers import ROOT, TINY, Oracle, RoundingJudge, random_tokens
from test_generate_gpu import check_greedy_path

pytestmark = pytest.mark.gpu

GROUPS = {"tiny_a": 64, "tiny_b": 32, "tiny_c": 64, "tiny_d": 128}


def engine(folder, name, **kw):
    from velox_b200 import Engine, EngineConfig
    kw.setdefault("weight_bits", 4)
    return Engine(folder, EngineConfig(page_size=TINY[name]["page_size"], max_model_len=kw.pop("max_model_len", 256), num_pages=kw.pop("num_pages", 128),
                                       weight_group=GROUPS[name], **kw), poison_cache=True)


def four_bits(w, name, head):
    """The plain implementation's weights with the layers' matrices (and the head) as their codes stand for them."""
    out = dict(w)
    for key, t in w.items():
        if key.endswith("_proj.weight") or (head and key == "lm_head.weight"):
            out[key] = q4.matrix(*q4.quantise(t.astype(np.float32), GROUPS[name]), GROUPS[name])
    return out


@pytest.mark.parametrize("name", ["tiny_a", "tiny_b", "tiny_c", "tiny_d"])
@pytest.mark.parametrize("head", [False, True])
def test_logits(model_folders, name, head):
    """Prompts of 1 to 150 tokens in one step each way, then decoded tokens: every row of logits."""
    from velox_b200.engine import StepEntry
    cfg, w = P.load_model_folder(model_folders[name])
    tied = cfg["tie_word_embeddings"]
    plain = four_bits(w, name, head)
    if head and tied:   # (the head takes a copy of the table in four bits, the embedding's stays)
        plain["lm_head.weight"] = q4.matrix(*q4.quantise(w["model.embed_tokens.weight"].astype(np.float32), GROUPS[name]), GROUPS[name])
        cfg = dict(cfg, tie_word_embeddings=False)
    e = engine(model_folders[name], name, head_bits=4 if head else None)
    assert e.model.blocks[0].mixer.qkv.matrix.group == GROUPS[name] and (e.model.head.q4 is not None) == head
    lens = (1, 5, 17, 40, 150)
    seqs = [random_tokens(cfg["vocab_size"], n + 4, 7 + n) for n in lens]
    oracles = [Oracle(cfg, plain, s) for s in seqs]
    judge = RoundingJudge.of(oracles, "four bits, %s" % name)
    for i in range(len(seqs)):
        e.cache.add_request(i)
    entries = [StepEntry(i, s[:n], want=list(range(n))) for i, (s, n) in enumerate(zip(seqs, lens))]
    got = e.run_step(entries).double().cpu().numpy()
    at = 0
    for o, n in zip(oracles, lens):
        judge.check(got[at:at + n], o.exact[:n], o.cost[:n], "prompt of %d" % n)
        at += n
    for k in range(4):
        got = e.run_step([StepEntry(i, [s[n + k]], want=[0]) for i, (s, n) in enumerate(zip(seqs, lens))]).double().cpu().numpy()
        judge.check(got, np.stack([o.exact[n + k] for o, n in zip(oracles, lens)]), np.array([o.cost[n + k] for o, n in zip(oracles, lens)]), "decoded %d" % k)
    judge.finish()


@pytest.mark.parametrize("name", ["tiny_b", "tiny_d"])
def test_generation_with_and_without_graphs(model_folders, name):
    """A run as a user has it: portions, mixed steps, captured decode steps; the cutting of prompts and the capture change nothing that
    the greedy path could not change by rounding."""
    from velox_b200 import SamplingParams
    cfg, w = P.load_model_folder(model_folders[name])
    plain = four_bits(w, name, False)
    prompts = [random_tokens(cfg["vocab_size"], n, 30 + n) for n in (3, 70, 21, 1)]
    for graphs in (True, False):
        e = engine(model_folders[name], name, cuda_graphs=graphs, chunk_size=33)
        outs = e.generate(prompts, SamplingParams(max_tokens=10))
        assert [len(o) for o in outs] == [10] * 4
        for p, o in zip(prompts, outs):
            check_greedy_path(cfg, plain, p, o, "bfloat16")
        e.cache.check()


def test_many_requests_decode_on_the_tensor_cores(model_folders):
    """20 requests decode side by side: more rows than the few that stream the matrices, captured, with bounded waits that are checked."""
    from velox_b200 import SamplingParams
    from velox_b200.csrc import ops
    cfg, w = P.load_model_folder(model_folders["tiny_c"])
    plain = four_bits(w, "tiny_c", False)
    e = engine(model_folders["tiny_c"], "tiny_c", max_running_requests=32)
    prompts = [random_tokens(cfg["vocab_size"], 2 + i, 500 + i) for i in range(20)]
    before = ops.bounded_wait_launches()
    outs = e.generate(prompts, SamplingParams(max_tokens=6))
    assert ops.bounded_wait_launches() > before and not ops.bounded_wait_pending()
    for p, o in zip(prompts, outs):
        check_greedy_path(cfg, plain, p, o, "bfloat16")


def test_a_decode_step_of_few_requests_waits_for_nothing(model_folders):
    from velox_b200.csrc import ops
    from velox_b200.engine import StepEntry
    e = engine(model_folders["tiny_c"], "tiny_c", cuda_graphs=False)
    e.cache.add_request(0)
    e.run_step([StepEntry(0, [1, 2, 3], want=[2])])
    before = ops.bounded_wait_launches()
    e.run_step([StepEntry(0, [4], want=[0])])
    assert ops.bounded_wait_launches() == before


def test_random_weights_and_memory():
    """Matrices made on the device are taken to four bits one part at a time; the layers hold what their codes need."""
    from velox_b200 import Engine, EngineConfig, Qwen3Config, SamplingParams
    cfg = Qwen3Config.from_dict(dict(TINY["tiny_d"]["config"], hidden_size=1024, intermediate_size=2048, num_hidden_layers=3))
    e = Engine(None, EngineConfig(weight_bits=4, weight_group=64, num_pages=64, max_model_len=128), model_config=cfg, random_seed=5)
    for b in e.model.blocks:
        n = sum(m.nbytes for m in (b.mixer.qkv.matrix, b.mixer.out.matrix, *b.feed_forward.pair, b.feed_forward.down.matrix))
        elements = 1024 * (8 * 128 + 512) + 3 * 1024 * 2048
        assert n == elements * (1 / 2 + 4 / 64)
        assert b.feed_forward.gate_up is None
    outs = e.generate([[1, 2, 3], [4] * 50], SamplingParams(max_tokens=4))
    assert [len(o) for o in outs] == [4, 4]


def test_refusals(model_folders):
    from velox_b200 import Engine, EngineConfig
    with pytest.raises(ValueError, match="rows of 96 do not go into four-bit groups of 64"):
        Engine(model_folders["tiny_b"], EngineConfig(page_size=8, num_pages=16, max_model_len=64, weight_bits=4, weight_group=64))
    import dobepel_helpers
    import tempfile
    with tempfile.TemporaryDirectory() as tmp:
        cfg = dobepel_helpers.CONFIGS["even"]
        folder = dobepel_helpers.write_model(tmp, cfg, dobepel_helpers.lively_weights(cfg, 15))
        with pytest.raises(ValueError, match="weight_bits=4: .* hold their matrices in the engine's element type only"):
            Engine(folder, EngineConfig(num_pages=16, max_model_len=64, weight_bits=4, weight_group=32))


def test_the_command_line(model_folders):
    import json
    import subprocess
    import sys
    out = subprocess.run([sys.executable, ROOT + "/bin/velox", "generate", "--model-dir", model_folders["tiny_c"], "--prompt-tokens", "1,2,3", "--max-tokens",
                          "4", "--weight-bits", "4", "--head-bits", "4", "--num-pages", "16", "--max-model-len", "64"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert len(json.loads(out.stdout.splitlines()[0])["tokens"]) == 4


@pytest.mark.parametrize("requests,waiting", [(40, 9), (20, 0)])
def test_replayed_decode_steps_of_many_requests(model_folders, requests, waiting):
    """40 requests: all nine products of a captured decode step run on the tensor cores' kernel, and each replay says so; 20 requests stream these small
    matrices, and no replay has anything to be checked."""
    from velox_b200 import SamplingParams
    from velox_b200.csrc import ops
    cfg, w = P.load_model_folder(model_folders["tiny_c"])
    e = engine(model_folders["tiny_c"], "tiny_c", max_running_requests=64, head_bits=4)
    prompts = [random_tokens(cfg["vocab_size"], 2 + i % 5, 900 + i) for i in range(requests)]
    ids = [e.add_request(p, SamplingParams(max_tokens=7)) for p in prompts]
    e.step()
    assert all(len(e.request(i).generated) == 1 for i in ids)
    counts = []
    while e.scheduler.has_work():
        before = ops.bounded_wait_launches()
        e.step()
        counts.append(ops.bounded_wait_launches() - before)
        assert not ops.bounded_wait_pending()
    assert len(counts) == 6 and counts[1:] == [waiting] * 5   # (the first of them is recorded)
    graphs = list(e.runner.graphs.graphs.values())
    assert len(graphs) == 1 and graphs[0].graph is not None and graphs[0].bounded_wait_launches == waiting
    plain = four_bits(w, "tiny_c", True)
    for p, i in zip(prompts, ids):
        check_greedy_path(cfg, plain, p, list(e.scheduler.finished[i].generated), "bfloat16")
