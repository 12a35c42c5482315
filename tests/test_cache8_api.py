"""Host side of the calls over caches in 8 bits, and of stretched rotary axes, without a GPU: what is refused and with which words, that
unusual but allowed tensors reach the kernels with the right numbers, layouts of structures, and the C interface's own refusals.

The tensors are fakes on "cuda:0": sizes, types and strides, no memory, so that nothing can be launched."""
from __future__ import annotations

import copy
import ctypes
import math
import pickle
import re
import shutil
import subprocess
import warnings
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from min_fa3_demo_b200 import _cabi, build, cache, min_fa3_op as op, rotary

warnings.filterwarnings("ignore", message="Accessing the data pointer of FakeTensor")
E4M3, F32 = torch.float8_e4m3fn, torch.float32
MODE = FakeTensorMode()
AXES = rotary.RotaryAxes.from_sections((16, 24, 24))


class Launched(Exception):
    pass


class Library:
    """Stands for the C library: keeps a call's arguments and goes no further."""

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *sizes: 1 << 16

        def call(args, scales, *more):
            struct = {"b2a_cache8_append": _cabi.AppendArgs, "b2a_tree8_fwd": _cabi.TreeArgs}[name]
            raise Launched(struct.from_buffer_copy(args), _cabi.CacheScales.from_buffer_copy(scales))
        return call


@pytest.fixture(params=["device known", "device new"])
def fake(request, monkeypatch):
    monkeypatch.setattr(op, "_SM100", {0} if request.param == "device known" else set())
    monkeypatch.setattr(cache, "_SM100", op._SM100)
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda device=None: (10, 0))
    monkeypatch.setattr(_cabi, "load", lambda lib=Library(): lib)
    monkeypatch.setattr(cache, "_on_device", lambda device: op._HERE)
    monkeypatch.setattr(cache, "_stream_ptr", lambda device: 0)
    monkeypatch.setattr(cache, "_tree_bytes", lambda *sizes: (1 << 16, 0))
    with MODE:
        yield


def t(*shape, dtype=torch.bfloat16, device="cuda:0"):
    return torch.empty(shape, dtype=dtype, device=device)


def i32(*shape):
    return t(*shape, dtype=torch.int32)


def f8(*shape):
    return t(*shape, dtype=E4M3)


def f32(*shape, device="cuda:0"):
    return t(*shape, dtype=F32, device=device)


def arguments(call):
    pages = dict(k_cache=f8(9, 32, 2, 128), v_cache=f8(9, 32, 2, 128), cache_lens=i32(3), block_table=i32(3, 4),
                 k_scales=f32(9, 2, 2), v_scales=f32(9, 2, 2))
    if call == "append":
        return dict(k=t(3, 5, 2, 128), v=t(3, 5, 2, 128), **pages, q=t(3, 5, 4, 128), positions=i32(3, 3, 5), axes=AXES)
    if call == "append packed":
        return dict(k=t(11, 2, 128), v=t(11, 2, 128), **pages, cu_seqlens=i32(4), q=None, positions=None, axes=None)
    if call == "tree":
        return dict(q=t(3, 5, 4, 128), **pages, tree_mask=t(3, 5, 5, dtype=torch.bool), max_seqlen_q=None, cu_seqlens_q=None, out=None)
    return dict(q=t(11, 4, 128), **pages, tree_mask=t(11, 6, dtype=torch.bool), max_seqlen_q=6, cu_seqlens_q=i32(4), out=None)


FUNCTIONS = {"append": cache.append_cache, "append packed": cache.append_cache, "tree": cache.forward_tree,
             "tree packed": cache.forward_tree}


def launch(call, **change):
    with pytest.raises(Launched) as caught:
        FUNCTIONS[call](**dict(arguments(call), **change))
    return caught.value.args


# ---------------------------------------------------------------------------------------
# Calls
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("call", list(FUNCTIONS))
def test_calls_in_order_reach_the_library(fake, call):
    args, scales = launch(call)
    view = args.cache
    assert (view.pages, view.page_size, view.heads_k, view.table_width, view.table_stride) == (9, 32, 2, 4, 4)
    assert list(view.k_stride) == [8192, 256, 128] and args.batch == 3
    assert scales.block == 16 and list(scales.k_stride) == [4, 2, 1] and list(scales.v_stride) == [4, 2, 1]
    if call == "append":
        assert (args.seqlen, args.total, args.heads_q) == (5, 15, 4)


@pytest.mark.parametrize("call", ["append", "tree"])
@pytest.mark.parametrize("size,blocks,block", [(32, 1, 32), (64, 2, 32), (64, 1, 64), (128, 1, 128), (256, 2, 128), (48, 3, 16)])
def test_slots_of_a_scale_with_pages(fake, call, size, blocks, block):
    _, scales = launch(call, k_cache=f8(9, size, 2, 128), v_cache=f8(9, size, 2, 128), k_scales=f32(9, blocks, 2),
                       v_scales=f32(9, blocks, 2))
    assert scales.block == block


@pytest.mark.parametrize("call", ["append", "tree"])
@pytest.mark.parametrize("size,blocks,block", [(1, 1, 16), (100, 7, 16), (100, 4, 32), (100, 2, 64), (100, 1, 128), (1001, 8, 128)])
def test_slots_of_a_scale_without_pages(fake, call, size, blocks, block):
    args, scales = launch(call, k_cache=f8(3, size, 2, 128), v_cache=f8(3, size, 2, 128), k_scales=f32(3, blocks, 2),
                          v_scales=f32(3, blocks, 2), block_table=None)
    assert scales.block == block and args.cache.page_size == size and not args.cache.block_table


def test_unusual_tensors_reach_the_library(fake):
    # Views of one pool: k and v side by side, their scales likewise, heads before slots; scales expanded where they are only read.
    pool, both = f8(9, 2, 2, 32, 128), f32(9, 2, 2, 2)
    heads = dict(k_cache=pool[:, 0].transpose(1, 2), v_cache=pool[:, 1].transpose(1, 2), k_scales=both[:, 0].transpose(1, 2),
                 v_scales=both[:, 1].transpose(1, 2))
    for call in FUNCTIONS:
        args, scales = launch(call, **heads)
        assert list(args.cache.k_stride) == [16384, 128, 4096] and list(scales.v_stride) == [8, 1, 2]
    for call in ("tree", "tree packed"):
        _, scales = launch(call, k_scales=f32(1, 1, 1).expand(9, 2, 2), v_scales=f32(1, 1, 2).expand(9, 2, 2))
        assert list(scales.k_stride) == [0, 0, 0] and list(scales.v_stride) == [0, 0, 1]
    # A dimension of one, whose stride nobody looks at.
    one = dict(k_cache=f8(9, 16, 2, 128), v_cache=f8(9, 16, 2, 128), k_scales=f32(9, 2).unsqueeze(1), v_scales=f32(9, 1, 2).expand(9, 1, 2))
    for call in FUNCTIONS:
        assert launch(call, **one)[1].block == 16


def test_nothing_is_launched_for_no_tokens(fake):
    a = arguments("append")
    assert cache.append_cache(**dict(a, k=t(3, 0, 2, 128), v=t(3, 0, 2, 128), q=None, positions=None, axes=None)) is None
    out, lse = cache.forward_tree(**dict(arguments("tree packed"), q=t(0, 4, 128), tree_mask=None), return_lse=True)
    assert out.shape == (0, 4, 128) and lse.shape == (4, 0)


together = "a cache of dtype torch.float8_e4m3fn and k_scales and v_scales go together"
shape = "must have shape [9, blocks, 2] with blocks of 16, 32, 64 or 128 of 32 slots, which they divide. Got "
REFUSALS = [(call, change, words) for call in FUNCTIONS for change, words in [
    (dict(k_scales=lambda: None, v_scales=lambda: None), together), (dict(k_scales=lambda: None), together),
    (dict(v_scales=lambda: None), together),
    (dict(k_cache=lambda: t(9, 32, 2, 128), v_cache=lambda: t(9, 32, 2, 128)), "k_cache must have dtype torch.float8_e4m3fn"),
    (dict(v_cache=lambda: t(9, 32, 2, 128)), "v_cache must have dtype torch.float8_e4m3fn"),
    (dict(k_cache=lambda: t(9, 32, 2, 128, dtype=torch.float8_e5m2)), "k_cache must have dtype torch.float8_e4m3fn"),
    (dict(v_cache=lambda: f8(9, 32, 3, 128)), "k_cache and v_cache must have the same shape"),
    (dict(k_cache=lambda: f8(9, 32, 2, 136)[..., :128]), "k_cache must be 16-byte aligned"),
    (dict(k_cache=lambda: f8(9, 32, 2, 64)), "k_cache must have head_dim D=128"),
    (dict(k_cache=lambda: f8(1, 32, 2, 128).expand(9, -1, -1, -1)), "k_cache must not be expanded"),
    (dict(k_scales=lambda: f32(9, 2, 2, device="cpu")), "k_scales must be on the same CUDA device"),
    (dict(v_scales=lambda: f32(9, 2, 2, device="cuda:1")), "v_scales must be on the same CUDA device"),
    (dict(v_scales=lambda: t(9, 2, 2)), "v_scales must have dtype torch.float32"),
    (dict(k_scales=lambda: f32(9, 2)), "k_scales " + shape + "[9, 2]"),
    (dict(k_scales=lambda: f32(8, 2, 2)), "k_scales " + shape + "[8, 2, 2]"),
    (dict(k_scales=lambda: f32(9, 2, 1)), "k_scales " + shape + "[9, 2, 1]"),
    (dict(v_scales=lambda: f32(9, 3, 2)), "v_scales " + shape + "[9, 3, 2]"),
    (dict(v_scales=lambda: f32(9, 32, 2)), "v_scales " + shape + "[9, 32, 2]"),
    (dict(v_scales=lambda: f32(9, 1, 2)), "k_scales and v_scales must have the same shape"),
    (dict(k_cache=lambda: f8(9, 24, 2, 128), v_cache=lambda: f8(9, 24, 2, 128)), "of 24 slots, which they divide. Got [9, 2, 2]"),
]] + [(call, change, words) for call in ("append", "append packed") for change, words in [
    (dict(k_scales=lambda: f32(1, 2, 2).expand(9, -1, -1)), "k_scales must not be expanded"),
    (dict(v_scales=lambda: f32(9, 2, 1).expand(-1, -1, 2)), "v_scales must not be expanded"),
]]


@pytest.mark.parametrize("call,change,words", REFUSALS, ids=[f"{c}-{w[:40]}-{n}" for n, (c, _, w) in enumerate(REFUSALS)])
def test_refusals(fake, call, change, words):
    given = arguments(call)
    given.update((name, make()) for name, make in change.items())
    with pytest.raises(RuntimeError, match=re.escape(words)):
        FUNCTIONS[call](**given)


def test_other_calls_refuse_8_bits(fake):
    pages = dict(k_cache=f8(9, 32, 2, 128), cache_lens=i32(3), weights=f32(3, 2, 128), block_table=i32(3, 4))
    with pytest.raises(RuntimeError, match="k_cache must have dtype torch.bfloat16"):
        cache.cache_weights(t(3, 5, 4, 128), lse=f32(3, 4, 5), **pages)
    with pytest.raises(RuntimeError, match="k_cache must have dtype torch.bfloat16"):
        cache.evict_cache(v_cache=f8(9, 32, 2, 128), budget=40, recent=8, **pages)


# ---------------------------------------------------------------------------------------
# The C interface
# ---------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    build.build()
    return _cabi.load()


def test_layout(tmp_path):
    gcc = shutil.which("gcc") or shutil.which("cc")
    if gcc is None:
        pytest.skip("no C compiler")
    header = Path(build.PKG_DIR).parent / "include" / "b200attn.h"
    names = [field[0] for field in _cabi.CacheScales._fields_]
    src = tmp_path / "sizes.c"
    offsets = "".join(f'printf(" %zu", offsetof(b2a_cache_scales, {name}));' for name in names)
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{header}"\nint main(void) {{ printf("%zu %zu",'
                   f' sizeof(b2a_cache_scales), offsetof(b2a_rotary_axes, magnitude)); {offsets} return 0; }}\n')
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", str(src), "-o", str(tmp_path / "sizes")], check=True)
    size, magnitude, *at = map(int, subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split())
    assert size == ctypes.sizeof(_cabi.CacheScales) == _cabi.SCALES.size and magnitude == _cabi.RotaryAxes.magnitude.offset
    assert at == [getattr(_cabi.CacheScales, name).offset for name in names]
    s = _cabi.CacheScales.from_buffer_copy(_cabi.SCALES.pack(*range(1, 10)))
    assert (s.k, s.v, list(s.k_stride), list(s.v_stride), s.block) == (1, 2, [3, 4, 5], [6, 7, 8], 9)


def filled(struct, **fields):
    args = struct()
    for name, value in fields.items():
        if isinstance(value, tuple):
            getattr(args, name)[:] = value
        else:
            setattr(args, name, value)
    return args


def c_call(lib, name, scales=None, cache_fields=None, **change):
    view = dict(k=256, v=256, block_table=256, table_stride=4, k_stride=(8192, 256, 128), v_stride=(8192, 256, 128), pages=9,
                page_size=32, heads_k=2, table_width=4)
    given = dict(k=256, v=256, k_stride=(4, 2, 1), v_stride=(4, 2, 1), block=16)
    given.update(scales or {})
    common = dict(cache=filled(_cabi.Cache, **dict(view, **(cache_fields or {}))), cache_lens=256, batch=3, workspace=256,
                  workspace_bytes=1 << 30)
    if name == "b2a_cache8_append":
        fields = dict(common, k=256, v=256, k_stride=(1280, 256, 128), v_stride=(1280, 256, 128), seqlen=5, total=15)
        fields.update(change)
        args = filled(_cabi.AppendArgs, **fields)
        return lib.b2a_cache8_append(ctypes.byref(args), ctypes.byref(filled(_cabi.CacheScales, **given)), None)
    fields = dict(common, q=256, out=256, lse=256, q_stride=(512, 128), seqlen_q=5, total_q=15, heads_q=4)
    scratch, size = change.pop("scratch", 256), change.pop("scratch_bytes", 1 << 40)
    fields.update(change)
    args = filled(_cabi.TreeArgs, **fields)
    return lib.b2a_tree8_fwd(ctypes.byref(args), ctypes.byref(filled(_cabi.CacheScales, **given)), scratch, size, None)


C_REFUSALS = [(name, change, words) for name in ("b2a_cache8_append", "b2a_tree8_fwd") for change, words in [
    (dict(scales=dict(k=0)), "the scales of the cache must not be NULL"),
    (dict(scales=dict(v=0)), "the scales of the cache must not be NULL"),
    *[(dict(scales=dict(block=n)), f"a scale must have 16, 32, 64 or 128 slots, got {n}") for n in (0, 8, 24, 256, -16)],
    (dict(scales=dict(block=64)), "page_size must be a multiple of a scale's slots, got 32 and 64"),
    (dict(scales=dict(k_stride=(4, -2, 1))), "strides of the scales must not be negative"),
    (dict(cache_fields=dict(k_stride=(8192, 264, 128))), "strides of a cache in 8 bits must be multiples of 16 elements"),
    (dict(cache_fields=dict(v=8)), "the cache must be 16-byte aligned"), (dict(cache_fields=dict(pages=0)), "must be positive"),
    (dict(batch=0), "must be"),
]] + [
    ("b2a_cache8_append", dict(cache_lens=0), "cache_lens must not be NULL"), ("b2a_cache8_append", dict(total=14), "total = batch * seqlen"),
    ("b2a_cache8_append", dict(q=256, heads_q=4), "q is turned by positions, so it needs axes"),
    ("b2a_cache8_append", dict(workspace=0), "workspace must be a 16-byte aligned"),
    ("b2a_tree8_fwd", dict(out=0), "out must be a 16-byte aligned"), ("b2a_tree8_fwd", dict(heads_q=3), "heads_q % heads_k must be 0"),
    ("b2a_tree8_fwd", dict(q_stride=(512, 100)), "strides of q must be multiples of 8 elements"),
    ("b2a_tree8_fwd", dict(scratch=8), "scratch must be a 16-byte aligned"),
    ("b2a_tree8_fwd", dict(scratch=None), "scratch must be a 16-byte aligned"),
    ("b2a_tree8_fwd", dict(workspace=0), "workspace must be a 16-byte aligned"),
]


@pytest.mark.parametrize("name,change,words", C_REFUSALS, ids=[f"{n}-{w[:30]}-{i}" for i, (n, _, w) in enumerate(C_REFUSALS)])
def test_refusals_of_the_c_interface(lib, name, change, words):
    assert c_call(lib, name, **change) == _cabi.B2A_ERR_INVALID_ARGUMENT
    assert words in _cabi.last_error()


@pytest.mark.parametrize("args,scales", [(True, False), (False, True), (False, False)])
def test_null_arguments(lib, args, scales):
    s = ctypes.byref(_cabi.CacheScales()) if scales else None
    assert lib.b2a_cache8_append(ctypes.byref(_cabi.AppendArgs()) if args else None, s, None) == _cabi.B2A_ERR_INVALID_ARGUMENT
    assert "args and scales must not be NULL" in _cabi.last_error()
    assert lib.b2a_tree8_fwd(ctypes.byref(_cabi.TreeArgs()) if args else None, s, None, 0, None) == _cabi.B2A_ERR_INVALID_ARGUMENT
    assert "args and scales must not be NULL" in _cabi.last_error()


# ---------------------------------------------------------------------------------------
# Stretched axes
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("factor,length,slow,fast", [(1, 4096, 1, 32), (4, 4096, 1, 32), (8, 8192, 1, 4), (2.5, 300, 0, 7.5),
                                                     (16, 100, 3, 3), (4, 4096, math.inf, math.inf), (4, 4096, 0, 0)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_stretched_frequencies(factor, length, slow, fast, adjacent):
    plain = rotary.RotaryAxes.from_sections((16, 24, 24), 1e6, adjacent=adjacent)
    long = plain.stretched(factor, length, slow=slow, fast=fast)
    assert (long.pairs, long.axes, long._c.adjacent) == (64, 3, int(adjacent)) and list(long._c.axis) == list(plain._c.axis)
    for i in range(64):
        f = 1e6 ** (-i / 64)
        wavelength = 2 * math.pi / f                    # in positions
        if length <= slow * wavelength:                 # few turns: positions as if they were `factor` times nearer together
            expected = f / factor
        elif length >= fast * wavelength:
            expected = f
        else:
            share = (length / wavelength - slow) / (fast - slow)
            expected = f / factor * (1 - share) + f * share
        # 64-bit roundings of a handful of operations, in units of 2^-64 of a turn.
        assert abs(long._c.turn[i] - rotary._turn(expected)) <= 16 * 2.0**-53 * f / (2 * math.pi) * 2**64 + 1
    assert long.magnitude == ctypes.c_float(0.1 * math.log(factor) + 1).value == long._c.magnitude


def test_stretched_magnitudes_and_what_is_as_before():
    plain = rotary.RotaryAxes.from_sections((64,), 1e4)
    assert plain.magnitude == 1.0 and plain.stretched(1, 100).magnitude == 1.0
    assert list(plain.stretched(1, 100)._c.turn) == list(plain._c.turn)
    assert plain.stretched(8, 100, magnitude=1).magnitude == 1.0 and plain.stretched(8, 100, magnitude=0.5).magnitude == 0.5
    twice = plain.stretched(2, 100).stretched(2, 200)
    assert abs(twice.magnitude - (0.1 * math.log(2) + 1) ** 2) < 4 * 2.0**-24
    assert rotary.RotaryAxes([0.5] * 8, magnitude=1.25).magnitude == 1.25
    zero = rotary.RotaryAxes([0.0, -0.25] * 4).stretched(4, 1000, slow=1, fast=2)
    assert list(zero._c.turn)[:2] == [0, rotary._turn(-0.25)]                # a negative frequency turns as often


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda a: pickle.loads(pickle.dumps(a))])
def test_copies_keep_what_they_are(how):
    axes = rotary.RotaryAxes.from_sections((16, 24, 24), 1e6, adjacent=True).stretched(4, 8192)
    other = how(axes)
    assert bytes(other._c) == bytes(axes._c) and other.magnitude == axes.magnitude and other._plain == axes._plain
    assert bytes(other.stretched(2, 100)._c) == bytes(axes.stretched(2, 100)._c)
    back = rotary.RotaryAxes._from_plain(*axes._plain, axes.magnitude)
    assert bytes(back._c) == bytes(axes._c)
    with pytest.raises(RuntimeError, match="do not know their frequencies"):
        back.stretched(2, 100)


@pytest.mark.parametrize("given,words", [
    (dict(factor=0.5), "factor must be 1 or more, got 0.5"), (dict(factor=math.nan), "factor must be"), (dict(factor=math.inf), "factor must be"),
    (dict(original_length=0), "original_length must be positive, got 0"), (dict(original_length=math.nan), "original_length must be positive"),
    (dict(slow=-1), "slow must be between 0 and fast. Got -1 vs 32"), (dict(slow=33), "Got 33 vs 32"), (dict(fast=math.nan), "slow must be"),
    (dict(magnitude=0.0), "magnitude must be positive and finite"), (dict(magnitude=-1.0), "magnitude must be positive and finite"),
    (dict(magnitude=math.nan), "magnitude must be"), (dict(magnitude=1e39), "magnitude must be positive and finite, got inf"),
])
def test_stretches_that_are_refused(given, words):
    with pytest.raises(RuntimeError, match=re.escape(words)):
        rotary.RotaryAxes.from_sections((64,)).stretched(**dict(dict(factor=4, original_length=4096), **given))


def test_magnitude_of_the_c_interface(lib):
    axes = rotary.RotaryAxes.from_sections((64,))
    axes._c.magnitude = math.inf
    args = filled(_cabi.RotaryArgs, axes=axes._at, q=256, q_out=256, positions=256, q_stride=(2560, 512, 128), positions_stride=(15, 5, 1),
                  batch=3, seqlen=5, heads_q=4)
    assert lib.b2a_rotary(ctypes.byref(args), None) == _cabi.B2A_ERR_INVALID_ARGUMENT and "magnitude must be finite" in _cabi.last_error()


@pytest.mark.parametrize("how", [lambda a: a, copy.copy, copy.deepcopy, lambda a: pickle.loads(pickle.dumps(a)),
                                 lambda a: rotary.RotaryAxes._from_plain(*a._plain, a.magnitude)])
def test_the_magnitude_is_the_same_for_all_calls(how):
    """The attribute is what traced steps read, the structure what kernels read."""
    axes = how(rotary.RotaryAxes([0.5] * 8, magnitude=1.25))
    with pytest.raises(AttributeError, match="magnitude cannot be changed"):
        axes.magnitude = 2.0
    assert axes.magnitude == axes._c.magnitude == 1.25


def test_which_types_a_call_says_it_takes(fake):
    """Calls without scales do not speak of them."""
    k8, v8, weights = f8(9, 32, 2, 128), f8(9, 32, 2, 128), f32(3, 2, 128)
    where = dict(cache_lens=i32(3), block_table=i32(3, 4))
    wide = dict(k_cache=t(9, 32, 2, 128), v_cache=t(9, 32, 2, 128), k_scales=None, v_scales=None)
    only = r"k_cache must have dtype torch\.bfloat16$"
    with pytest.raises(RuntimeError, match=only):
        cache.cache_weights(t(3, 5, 4, 128), f32(3, 4, 5), k8, weights=weights, **where)
    with pytest.raises(RuntimeError, match=only):
        cache.evict_cache(k8, v8, weights, budget=64, **where)
    for call, function in FUNCTIONS.items():
        with pytest.raises(RuntimeError, match=r"k_cache must have dtype torch\.bfloat16 or, with scales, torch\.float8_e4m3fn$"):
            function(**dict(arguments(call), **dict(wide, k_cache=t(9, 32, 2, 128, dtype=torch.float16))))
        with pytest.raises(RuntimeError, match=r"k_cache must have dtype torch\.float8_e4m3fn$"):
            function(**dict(arguments(call), k_cache=t(9, 32, 2, 128)))


@pytest.mark.parametrize("total,heads,stride", [(1, 4, (1001, 128)), (1, 2, (0, 256)), (15, 2, (512, 77)), (1, 1, (3, 5))])
def test_strides_that_nobody_looks_at_over_the_c_interface(lib, total, heads, stride):
    """One token, or one query head: as over a bf16 cache, the stride may be anything.  (Two heads of 15 tokens: it may not.)"""
    kvh = dict(cache_fields=dict(heads_k=1)) if heads == 1 else {}
    rc = c_call(lib, "b2a_tree8_fwd", batch=total // min(total, 5), seqlen_q=min(total, 5), total_q=total, heads_q=heads, q_stride=stride, **kvh)
    refused = rc == _cabi.B2A_ERR_INVALID_ARGUMENT and "strides of q" in _cabi.last_error()
    assert rc != _cabi.B2A_OK and refused == (total > 1)
