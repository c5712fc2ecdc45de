"""Models served from a cache held in 4 bits: the mixer against a plain computation over the stored numbers, whole engines,
replayed steps, the command line."""
import math
import subprocess
import sys

import pytest
import torch

import plain_kv4
from helpers import ROOT, TINY, make_folder, random_tokens

pytestmark = pytest.mark.gpu


def engine_for(folder, cache_dtype="int4", max_tokens=4096, block_size=64, graphs=True, max_batch=0):
    from stratakv_b200 import Engine, EngineConfig
    return Engine.from_folder(folder, EngineConfig(max_tokens=max_tokens, block_size=block_size, max_context=max_tokens, cache_dtype=cache_dtype,
                                                   use_cuda_graphs=graphs, max_batch=max_batch), verbose=False)


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("kv4")
    return {name: make_folder(root / name, TINY[name], seed=5, dtype="bfloat16") for name in TINY}


@pytest.mark.parametrize("name,block", [("A", 16), ("D", 64), ("E", 64), ("E", 48), ("C", 32), ("F", 16)])
def test_the_mixer_attends_over_what_it_stored(folders, name, block):
    """Prompts, single tokens and a few at once through one mixer: its result against 64 bits over the plain form's stored numbers of the
    very same projections."""
    from stratakv_b200 import StepEntry, ops
    engine = engine_for(folders[name], block_size=block)
    mixer = engine.model.layers[0].mixer
    s = mixer.spec
    assert s.cache_bits == 4 and engine.cache.entry_storage(0)["k"].dtype == torch.uint8
    slots = [engine.open_sequence() for _ in range(2)]
    before, stored = [0, 0], [[], []]
    for new in ([90, 33], [1, 1], [3, 1], [1, 1], [1, 70]):
        entries = [StepEntry(slot, [1] * c, []) for slot, c in zip(slots, new)]
        step, _, _ = engine.prepare(entries)
        n = sum(new)
        h = torch.randn(n, s.hidden_size, device="cuda").bfloat16()
        qkv = torch.empty(n, mixer.q_dim + 2 * mixer.kv_dim, device="cuda")
        engine.rt.kernels(s.head_dim).linear(h, mixer.w_qkv, qkv, ops.MODE_STORE_F32)
        x = torch.zeros(n, s.hidden_size, device="cuda")
        mixer.forward(step, h, x, 0, True)
        rows = qkv.view(n, -1, s.head_dim)
        turned = plain_kv4.rotate(rows[:, :s.num_heads + s.num_kv_heads], mixer.position.fusion_table(step.max_ctx), step.positions)
        ctx, allowed, at = [], [], 0
        for i, c in enumerate(new):
            mine = slice(at, at + c)
            stored[i].append([plain_kv4.read(*plain_kv4.store(part[mine])) for part in (turned[:, s.num_heads:], rows[:, s.num_heads + s.num_kv_heads:])])
            keys, values = (torch.cat([piece[j] for piece in stored[i]]).transpose(0, 1) for j in (0, 1))
            ref, sums, whole = plain_kv4.attention(turned[mine, :s.num_heads].bfloat16().double(), keys, values, before[i], s.scale)
            ctx.append(ref)
            # (rounded once; probabilities of 8 bits at worst, sums of products and exponentials 2^-11: see test_kv4_gpu.py)
            allowed.append(2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -11) * sums + 2.0 ** -32 * whole)
            at += c
            engine.cache.advance(slots[i], before[i] + c)
            before[i] += c
        w = mixer.w_o.double()
        ctx, allowed = (torch.cat(part).flatten(1) for part in (ctx, allowed))
        # the projection's own sums: at most heads * head_dim roundings of 2^-24, and the tensor core's cut of 2^-23 per product
        bound = allowed @ w.abs().T + 2.0 ** -22 * ctx.shape[1] ** 0.5 * (ctx.abs() @ w.abs().T) + 1e-30
        error = (x.double() - ctx @ w.T).abs()
        assert bool((error <= bound).all()), (new, float((error / bound).max()))


@pytest.mark.parametrize("name", ["A", "B", "E"])
def test_requests_end_to_end(folders, name):
    """Replayed and eager steps choose the same way over the same stored numbers, every block comes back, and the logits are those of the 16-bit
    cache but for what 4 bits lose."""
    from stratakv_b200 import StepEntry
    from stratakv_b200.sampling import SamplingParams
    vocab = TINY[name]["vocab_size"]
    prompts = [random_tokens(vocab, n, seed=n) for n in (33, 5, 61)]
    engines = {kind: engine_for(folders[name], kind if kind != "eager" else "int4", graphs=kind != "eager") for kind in ("int4", "eager", "")}
    logits = {}
    for kind, engine in engines.items():
        slots = [engine.open_sequence() for _ in prompts]
        got = [engine.step([StepEntry(slot, p[:-2], [len(p) - 3]) for slot, p in zip(slots, prompts)]).clone()]
        for i in (2, 1):
            got.append(engine.step([StepEntry(slot, [p[-i]], [0]) for slot, p in zip(slots, prompts)]).clone())
        logits[kind] = torch.cat(got).double()
        for slot in slots:
            engine.close_sequence(slot)
        engine.check_flags()
        assert engine.cache.all_free()
    assert engines["int4"].graph_launches > 0 and engines["eager"].graph_launches == 0
    spread = logits[""].std()
    # what rounding to steps of a seventh of a group's largest number does to a logit; a wrong key or position moves most logits by a
    # fraction of their spread
    assert float((logits["int4"] - logits[""]).std() / spread) < 0.35
    assert float((logits["int4"] - logits["eager"]).std() / spread) < 0.1
    out = engines["int4"].generate(prompts, 12, SamplingParams(temperature=0.8, top_k=20, seed=3), ignore_eos=True)
    again = engines["int4"].generate(prompts, 12, SamplingParams(temperature=0.8, top_k=20, seed=3), ignore_eos=True)
    assert out.sequences == again.sequences and [len(s) for s in out.sequences] == [len(p) + 12 for p in prompts]
    assert engines["int4"].cache.bytes_per_token() < 0.3 * engines[""].cache.bytes_per_token()


def test_a_sequence_is_alone_in_its_batch(folders):
    """The same tokens whoever else is in the step: batches of 1 and of 3, whose pieces of the context are cut alike or not."""
    engine = engine_for(folders["E"])
    prompts = [random_tokens(300, n, seed=n) for n in (40, 200, 7)]
    together = engine.generate(prompts, 20, ignore_eos=True).sequences
    for i, prompt in enumerate(prompts):
        alone = engine.generate([prompt], 20, ignore_eos=True).sequences[0]
        assert alone[:len(prompt) + 1] == together[i][:len(prompt) + 1]


def test_the_command_line(folders):
    command = [sys.executable, str(ROOT / "bin" / "stratakv_cli"), "--cache-dtype", "int4", str(folders["E"]), "5", "3", "1", "4"]
    result = subprocess.run(command, capture_output=True, text=True, timeout=300)
    assert result.returncode == 0, result.stderr
    assert len(result.stdout.split()) <= 8 and result.stdout.split()[:3] == ["3", "1", "4"]
    result = subprocess.run(command[:2] + ["--dtype", "float32"] + command[2:], capture_output=True, text=True, timeout=300)
    assert result.returncode == 1 and "bfloat16 kernels alone" in result.stderr


def windowed_engine(window, block_size, max_tokens):
    import dataclasses
    from stratakv_b200 import Engine, EngineConfig
    from stratakv_b200.config import LlamaConfig
    from stratakv_b200.config.registry import resolve_architecture
    from stratakv_b200.engine.model import expected_tensors
    from stratakv_b200.weights.random_init import random_tensors
    config = LlamaConfig.from_dict(TINY["E"])
    spec = resolve_architecture(config.architecture).build_spec(config)
    spec = dataclasses.replace(spec, layers=tuple(dataclasses.replace(layer, mixer=dataclasses.replace(layer.mixer, window=window)) for layer in spec.layers))
    tensors = random_tensors(expected_tensors(spec), 5, dtype=torch.bfloat16)
    return Engine(spec, tensors, EngineConfig(max_tokens=max_tokens, block_size=block_size, max_context=4096, cache_dtype="int4"), verbose=False)


@pytest.mark.parametrize("direct", [True, False])
@pytest.mark.parametrize("block", [16, 64])
def test_a_window_whose_blocks_others_take(monkeypatch, block, direct):
    """Two sequences through a windowed layer whose cache is so small that what the one's window gives back is the other's next: each attends over its
    own last positions alone.  ``direct``: prompts read the 4-bit cache too."""
    from stratakv_b200 import StepEntry, ops
    window = 40
    engine = windowed_engine(window, block, 224 if block == 16 else 384)
    monkeypatch.setattr(ops.Kernels, "_kv4_few", staticmethod(lambda n_seqs, max_q_len, *sizes: direct or max_q_len < 8))
    mixer = engine.model.layers[0].mixer
    s = mixer.spec
    assert s.cache_bits == 4 and s.window == window and engine.cache.groups[0].kind.name == "kv4_window"
    slots = [engine.open_sequence() for _ in range(2)]
    before, stored, had = [0, 0], [[], []], [set(), set()]
    for new in ([90, 20], [1, 1], [1, 60], [100, 1], [1, 100], [1, 1], [3, 2], [1, 1]):
        step, _, _ = engine.prepare([StepEntry(slot, [1] * c, []) for slot, c in zip(slots, new)])
        for i, slot in enumerate(slots):
            had[i] |= set(engine.cache.sequences[slot].blocks[0])
        n = sum(new)
        h = torch.randn(n, s.hidden_size, device="cuda").bfloat16()
        qkv = torch.empty(n, mixer.q_dim + 2 * mixer.kv_dim, device="cuda")
        engine.rt.kernels(s.head_dim).linear(h, mixer.w_qkv, qkv, ops.MODE_STORE_F32)
        x = torch.zeros(n, s.hidden_size, device="cuda")
        mixer.forward(step, h, x, 0, True)
        rows = qkv.view(n, -1, s.head_dim)
        turned = plain_kv4.rotate(rows[:, :s.num_heads + s.num_kv_heads], mixer.position.fusion_table(step.max_ctx), step.positions)
        ctx, allowed, at = [], [], 0
        for i, c in enumerate(new):
            mine = slice(at, at + c)
            stored[i].append([plain_kv4.read(*plain_kv4.store(part[mine])) for part in (turned[:, s.num_heads:], rows[:, s.num_heads + s.num_kv_heads:])])
            keys, values = (torch.cat([piece[j] for piece in stored[i]]).transpose(0, 1) for j in (0, 1))
            ref, sums, whole = plain_kv4.attention(turned[mine, :s.num_heads].bfloat16().double(), keys, values, before[i], s.scale, window)
            ctx.append(ref)
            # (rounded once; probabilities of 8 bits at worst, sums of products and exponentials 2^-11)
            allowed.append(2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -11) * sums + 2.0 ** -32 * whole)
            at += c
            engine.cache.advance(slots[i], before[i] + c)
            before[i] += c
        w = mixer.w_o.double()
        ctx, allowed = (torch.cat(part).flatten(1) for part in (ctx, allowed))
        # the projection's own sums: at most heads * head_dim roundings of 2^-24, and the tensor core's cut of 2^-23 per product
        bound = allowed @ w.abs().T + 2.0 ** -22 * ctx.shape[1] ** 0.5 * (ctx.abs() @ w.abs().T) + 1e-30
        error = (x.double() - ctx @ w.T).abs()
        assert bool((error <= bound).all()), (new, float((error / bound).max()))
    assert had[0] & had[1]


def test_decode_steps_keep_to_their_own_sequence(folders):
    """The same tokens given to sequences in a batch and to each alone: their logits differ by what another order of sums does to the stored codes.
    bfloat16 rows that differ by a rounding (2^-8 of a number) store another code where they straddle a border of codes: a step is a seventh of a
    group's largest number, so in up to 7 x 2^-8 of the numbers, 3 %, by a step each, 0.17 of a step in the mean square; the rounding to codes itself
    is 0.29 of a step.  So this is at most 0.6 of what 4 bits do to a logit, 0.35 of the logits' spread: 0.21.  Another sequence's keys move them by more."""
    from stratakv_b200 import StepEntry
    engine = engine_for(folders["E"])
    lengths = (40, 200, 7)
    prompts = [random_tokens(300, n, seed=n) for n in lengths]
    forced = [random_tokens(300, 12, seed=100 + n) for n in lengths]

    def logits_of(prompts, forced):
        slots = [engine.open_sequence() for _ in prompts]
        engine.step([StepEntry(slot, p, []) for slot, p in zip(slots, prompts)])
        got = torch.stack([engine.step([StepEntry(slot, [f[i]], [0]) for slot, f in zip(slots, forced)]).clone() for i in range(12)], dim=1).double()
        for slot in slots:
            engine.close_sequence(slot)
        engine.check_flags()
        return got

    launched = engine.graph_launches
    together = logits_of(prompts, forced)
    assert engine.graph_launches > launched
    for i, n in enumerate(lengths):
        alone = logits_of([prompts[i]], [forced[i]])[0]
        other = logits_of([random_tokens(300, n, seed=50 + n)], [forced[i]])[0]
        spread = float(alone.std())
        moved, told = float((together[i] - alone).std()) / spread, float((other - alone).std()) / spread
        print(f"length {n}: together {moved:.4f}, behind another prompt {told:.4f}")
        assert moved < 0.21
        assert told > 2 * moved
    assert engine.cache.all_free()
