"""A cache held in 4 bits without a GPU: its format, its storage, who may ask for it, and what the libraries refuse."""
import ctypes
import dataclasses
import math
import re

import pytest
import torch

import plain_kv4
from helpers import TINY
from stratakv_b200 import ConfigError, EngineConfig
from stratakv_b200.cache import KVCache
from stratakv_b200.config import LlamaConfig
from stratakv_b200.csrc import build
from stratakv_b200.parts.base import CacheRequest


def test_what_is_stored_is_near_and_exact_in_16_bits():
    x = torch.randn(200, 64, generator=torch.Generator().manual_seed(1)) * torch.logspace(-6, 3, 200)[:, None]
    codes, scale = plain_kv4.store(x)
    near = plain_kv4.read(codes, scale)
    step = plain_kv4.scale_table()[scale.long()].repeat_interleave(16, dim=-1)
    assert bool(((near - x.double()).abs() <= 0.5 * step * (1 + 2.0 ** -20)).all())
    for dtype in (torch.bfloat16, torch.float16):
        assert torch.equal(near.to(dtype).double(), near)
    table = plain_kv4.scale_table()[:plain_kv4.LARGEST + 1]
    assert bool((table.diff() > 0).all()) and float(table[-1] * 7) == 6272.0
    # 9/8 of a scale's half, which the kernels multiply by, is a half for every byte that is written
    assert torch.equal((table * 64 * 1.125).half().double(), table * 64 * 1.125)
    bad, byte = plain_kv4.store(torch.tensor([[1.0] * 15 + [math.inf], [math.nan] * 16, [0.0] * 16]))
    assert byte.tolist() == [[255], [255], [0]] and bool((bad == 0x88).all())
    assert bool(torch.isnan(plain_kv4.read(bad, byte)[:2]).all())


def test_storage_in_4_bits():
    requests = [CacheRequest("kv4", 2, 64), CacheRequest("kv", 2, 64), CacheRequest("kv4_window", 2, 32, 40)]
    cache = KVCache(requests, 6, 16, 3, torch.bfloat16, "cpu")
    stored = cache.entry_storage(0)
    assert {name: (tuple(t.shape), t.dtype) for name, t in stored.items()} == {
        "k": ((7, 2, 16, 32), torch.uint8), "v": ((7, 2, 16, 32), torch.uint8),
        "k_scale": ((7, 2, 16, 4), torch.uint8), "v_scale": ((7, 2, 16, 4), torch.uint8)}
    assert cache.entry_storage(1)["k"].dtype == torch.bfloat16
    assert cache.bytes_per_token() == 2 * 2 * 36 + 2 * 2 * 128 + 2 * 2 * 18
    # a window's blocks are given back as those of the 16-bit kind are
    slot = cache.acquire()
    cache.reserve({slot: 90})
    cache.advance(slot, 90)
    assert cache.sequences[slot].dropped[2] == (90 - 40 + 1) // 16 and cache.sequences[slot].dropped[0] == 0
    cache.release(slot)
    assert cache.all_free()


def test_configurations():
    assert EngineConfig(max_tokens=64).cache_dtype == "" and EngineConfig(max_tokens=64, cache_dtype="int4").cache_dtype == "int4"
    assert EngineConfig(max_tokens=64, dtype="float32", cache_dtype="float32").dtype == torch.float32
    for match, changes in (("bfloat16 kernels alone", dict(dtype="float32", cache_dtype="int4")), ("compute dtype or int4", dict(cache_dtype="float32")),
                           ("compute dtype must be", dict(cache_dtype="int3"))):
        with pytest.raises(ConfigError, match=match):
            EngineConfig(max_tokens=64, **changes)


def spec_of(name):
    config = LlamaConfig.from_dict(TINY[name])
    from stratakv_b200.config.registry import resolve_architecture
    return resolve_architecture(config.architecture).build_spec(config)


def test_the_engine_asks_for_it_layer_by_layer():
    from stratakv_b200.engine.engine import Engine
    from stratakv_b200.engine.model import cache_requests
    spec = spec_of("A")
    assert Engine._kept_in(spec, EngineConfig(max_tokens=64)) is spec
    kept = Engine._kept_in(spec, EngineConfig(max_tokens=64, cache_dtype="int4"))
    assert all(layer.mixer.cache_bits == 4 for layer in kept.layers) and all(layer.mixer.cache_bits == 0 for layer in spec.layers)
    assert {r.kind for r in cache_requests(kept)} == {"kv4"} and {r.kind for r in cache_requests(spec)} == {"kv"}
    windowed = dataclasses.replace(spec, layers=tuple(dataclasses.replace(layer, mixer=dataclasses.replace(layer.mixer, window=32)) for layer in spec.layers))
    assert {r.kind for r in cache_requests(Engine._kept_in(windowed, EngineConfig(max_tokens=64, cache_dtype="int4")))} == {"kv4_window"}
    capped = dataclasses.replace(spec, layers=(spec.layers[0], dataclasses.replace(spec.layers[1], mixer=dataclasses.replace(spec.layers[1].mixer, softcap=30.0))))
    with pytest.raises(ConfigError, match="plain attention"):
        Engine._kept_in(capped, EngineConfig(max_tokens=64, cache_dtype="int4"))


@pytest.mark.parametrize("module", ["zepavik", "povusun", "kedelorn", "fidolix", "tobozen", "vekanex"])
def test_models_with_other_layers_are_refused(module):
    import importlib
    from stratakv_b200.engine.engine import Engine
    from stratakv_b200.config.registry import resolve_architecture
    raw = next(iter(getattr(importlib.import_module(f"{module}_models"), module.upper()).values()))
    arch = resolve_architecture(raw["architecture"])
    with pytest.raises(ConfigError, match="4 bits"):
        Engine._kept_in(arch.build_spec(arch.config_class.from_dict(raw)), EngineConfig(max_tokens=64, cache_dtype="int4"))


def test_command_line():
    from stratakv_b200.cli import parse_arguments
    from stratakv_b200.runner import parse_args
    assert parse_arguments(["--cache-dtype", "int4", "m", "3", "1"]).cache_dtype == "int4"
    assert parse_arguments(["m", "3", "1"]).cache_dtype == ""
    assert parse_args(["--model", "m", "--cache-dtype", "int4"]).cache_dtype == "int4"


def library(dtype, head_dim):
    path = build.find_built(dtype, head_dim)
    if path is None:
        pytest.skip("not compiled yet")
    lib = ctypes.CDLL(str(path))
    lib.skv_last_error.restype = ctypes.c_char_p
    return lib


def test_the_libraries_refuse_bad_sizes():
    """Arguments that never reach a kernel: each is refused with its reason (no device is needed)."""
    lib = library("bfloat16", 64)
    null, i, odd = ctypes.c_void_p(0), ctypes.c_int, ctypes.c_void_p(8)

    def append(tokens=1, heads=4, kv=2, dim=64, block=16, qkv=null):
        code = lib.skv_append_kv4(qkv, null, null, null, null, i(1), null, null, null, null, null, i(tokens), i(heads), i(kv), i(dim), i(block),
                                  i(1), null)
        return code, lib.skv_last_error().decode()

    assert append(tokens=0)[0] == 0
    for match, changes in (("multiple of 16", dict(dim=40)), ("multiple of kv heads", dict(heads=5)), ("multiple of kv heads", dict(kv=0)),
                           ("block_size", dict(block=24)), ("aligned", dict(qkv=odd)), ("too long", dict(heads=2 ** 21, kv=1))):
        code, message = append(**changes)
        assert code != 0 and match in message, (changes, message)

    def unpack(seqs=1, width=1, kv=2, dim=64, block=16, keep=0, out=null):
        code = lib.skv_unpack_kv4(null, null, null, null, null, i(1), null, out, null, null, i(seqs), i(width), i(kv), i(dim), i(block), i(keep), null)
        return code, lib.skv_last_error().decode()

    assert unpack(seqs=0)[0] == 0 and unpack(width=0)[0] == 0
    for match, changes in (("multiple of 16", dict(dim=8)), ("block_size", dict(block=0)), ("kv heads", dict(kv=0)), ("must not be negative", dict(keep=-1)),
                           ("too many", dict(seqs=2 ** 20, width=2 ** 12)), ("aligned", dict(out=odd))):
        code, message = unpack(**changes)
        assert code != 0 and match in message, (changes, message)

    def attend(seqs=1, most=1, heads=4, kv=2, dim=64, block=16, window=0, q=null, width=1, floats=0, scratch=null):
        code = lib.skv_attention_kv4(q, null, null, null, null, null, i(width), null, null, null, scratch, ctypes.c_longlong(floats), i(seqs), i(most),
                                     i(heads), i(kv), i(dim), i(block), ctypes.c_float(1.0), i(window), null)
        return code, lib.skv_last_error().decode()

    assert attend(seqs=0)[0] == 0 and attend(width=0)[0] == 0 and attend(most=0)[0] == 0
    for match, changes in (("another head size", dict(dim=128)), ("multiple of kv heads", dict(heads=3)), ("block_size", dict(block=8)),
                           ("must not be negative", dict(window=-3)), ("aligned", dict(q=odd)), ("too many rows", dict(heads=64, kv=64, most=2 ** 25)),
                           ("too many positions", dict(width=2 ** 30)), ("too large", dict(kv=4, block=2 ** 27)), ("aligned", dict(scratch=odd))):
        code, message = attend(**changes)
        assert code != 0 and match in message, (changes, message)


def test_append_refuses_a_cache_that_no_reader_takes():
    """Codes are stored two bytes at a time, and read 16 bytes at a time."""
    lib = library("bfloat16", 64)
    null, i = ctypes.c_void_p(0), ctypes.c_int
    for which in range(4):
        cache = [ctypes.c_void_p(1 if of == which else 0) for of in range(4)]
        assert lib.skv_append_kv4(null, null, null, null, null, i(1), null, *cache, i(1), i(4), i(2), i(64), i(16), i(1), null) != 0
        assert b"aligned" in lib.skv_last_error()


def scratch_of(lib, seqs=1, most=1, width=4, heads=4, kv=2, block=16, window=0):
    lib.skv_attention_kv4_scratch.restype = ctypes.c_longlong
    return lib.skv_attention_kv4_scratch(*(ctypes.c_int(n) for n in (seqs, most, width, heads, kv, block, window)))


def test_scratch_of_sizes_that_are_refused():
    lib = library("bfloat16", 64)
    assert scratch_of(lib) > 0
    for changes in (dict(width=0), dict(width=-1), dict(block=8, width=1), dict(block=0), dict(block=24), dict(heads=3), dict(heads=0), dict(kv=0),
                    dict(seqs=0), dict(most=0), dict(window=-1)):
        assert scratch_of(lib, **changes) == 0, changes


def test_a_window_that_no_position_can_leave_is_none():
    lib = library("bfloat16", 64)
    for most in (1, 5, 300):
        for window in (64, 1000, 2 ** 31 - 1):
            assert scratch_of(lib, most=most, window=window) == scratch_of(lib, most=most) > 0


def test_float32_libraries_have_none():
    lib = library("float32", 64)
    null, i = ctypes.c_void_p(0), ctypes.c_int
    assert lib.skv_has_kv4() == 0 and library("bfloat16", 64).skv_has_kv4() == 1
    assert lib.skv_append_kv4(null, null, null, null, null, i(1), null, null, null, null, null, i(1), i(1), i(1), i(64), i(16), i(1), null) != 0
    assert b"bfloat16" in lib.skv_last_error()
    assert lib.skv_attention_kv4(null, null, null, null, null, null, i(1), null, null, null, null, ctypes.c_longlong(0), i(1), i(1), i(1), i(1), i(64),
                                 i(16), ctypes.c_float(1.0), i(0), null) != 0
    assert b"bfloat16" in lib.skv_last_error()


def without_lambdas(text):
    while (at := text.find("[&]")) >= 0:
        end = start = text.index("{", at)
        depth = 0
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        text = text[:at] + text[end:]
    return text


def test_no_kernel_leaves_ahead_of_its_wait():
    """A grid whose blocks all return before they wait for the grid in front of them is complete before that one, and whoever waits for it alone runs
    beside the other: attention over the next piece of a scratch, while the piece before is still written."""
    seen = 0
    for path in sorted(build.CSRC.glob("*.cu")):
        for piece in path.read_text().split("pdl_launch_dependents();")[1:]:
            body = without_lambdas(piece.split("\n}\n")[0])
            seen += 1
            assert "pdl_wait();" in body, path.name
            for leaving in re.finditer(r"\breturn;", body[:max(0, body.rfind("pdl_wait();"))]):
                before = body[:leaving.start()].rstrip()
                assert before.endswith("pdl_wait();") or before.count("pdl_wait();") > before.count("return;"), path.name
    assert seen > 50


def test_scratch_grows_within_its_bound(monkeypatch):
    """A buffer with a bound doubles up to it, takes what is asked for beyond, and is gone before the larger one is made."""
    import weakref
    from stratakv_b200.parts.workspace import Workspace
    made, real = [], torch.empty

    def empty(count, **options):
        assert all(old() is None for _, old in made)
        tensor = real(count, **options)
        made.append((count, weakref.ref(tensor)))
        return tensor

    workspace = Workspace("cpu")
    monkeypatch.setattr(torch, "empty", empty)
    for count in (100, 90, 150, 700, 1400, 1500, 1600, 1550, 3000, 20):
        assert workspace.get("scratch", (count,), torch.uint8, most=1600).numel() == count
    assert [count for count, _ in made] == [100, 200, 700, 1400, 1600, 3000] and workspace.generation == 6
    made.clear()
    for count in (100, 150, 250):                          # (without a bound: twice as much)
        workspace.get("rows", (count,), torch.float32)
    assert [count for count, _ in made] == [100, 200, 400]


def test_prompts_ask_for_scratch_within_its_bound():
    """What the mixer asks its workspace for: a bound of 1 GB beside the bytes of the step."""
    from types import SimpleNamespace
    from stratakv_b200 import ops
    from stratakv_b200.parts.attention import PagedAttention
    asked = {}

    def get(name, shape, dtype, zero=False, most=0):
        asked[name] = (shape, most)
        return torch.empty(shape, dtype=dtype)

    wanted = [3000]
    kernels = SimpleNamespace(append_kv4=lambda *a: None, attention_kv4=lambda *a: None, attention_kv4_scratch=lambda *a: wanted[0])
    cache = SimpleNamespace(block_size=64, entry_storage=lambda e: {"k": 0, "v": 0, "k_scale": 0, "v_scale": 0}, entry_group_index=lambda e: 0)
    step = SimpleNamespace(cache=cache, block_tables={0: torch.zeros(1, 5)}, max_ctx=300, positions=None, token_seq=None, n_seqs=1, max_q_len=300, cu_q=None,
                           ctx_after=None)
    mixer = SimpleNamespace(spec=SimpleNamespace(num_heads=4, num_kv_heads=2, head_dim=64, window=0, scale=0.125), q_dim=256,
                            rt=SimpleNamespace(kernels=lambda dim: kernels, dtype=torch.bfloat16, workspace=SimpleNamespace(get=get)),
                            position=SimpleNamespace(fusion_table=lambda n: None))
    PagedAttention._attend_in_4_bits(mixer, step, torch.zeros(300, 512), None, 0, True)
    assert asked["kv4_scratch"] == ((3000,), ops.KV4_UNPACKED)


def test_reading_back_what_is_seen_refuses_bad_sizes():
    lib = library("bfloat16", 64)
    null, i = ctypes.c_void_p(0), ctypes.c_int

    def seen(cu=ctypes.c_void_p(4), most=1, window=0, tile=64, seqs=1, width=1, dim=64, block=16, kv=2):
        code = lib.skv_unpack_kv4_seen(null, null, null, null, null, i(1), null, null, null, null, i(seqs), i(width), i(kv), i(dim), i(block), cu, i(most),
                                       i(window), i(tile), null)
        return code, lib.skv_last_error().decode()

    assert seen(seqs=0)[0] == 0 and seen(width=0, cu=null)[0] == 0
    for match, changes in (("offsets", dict(cu=null)), ("must not be negative", dict(most=-1)), ("must not be negative", dict(window=-1)), ("positive tile", dict(tile=0)),
                           ("multiple of 16", dict(dim=40)), ("block_size", dict(block=8)), ("kv heads", dict(kv=0)), ("too many", dict(seqs=2 ** 20, width=2 ** 12))):
        code, message = seen(**changes)
        assert code != 0 and match in message and "skv_unpack_kv4_seen" in message, (changes, message)
    assert library("float32", 64).skv_unpack_kv4_seen(*([null] * 5), i(1), *([null] * 4), i(1), i(1), i(1), i(64), i(16), null, i(1), i(0), i(64), null) != 0
