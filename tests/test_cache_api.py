"""Host side of the rotary and cache calls, without a GPU: what is exported, what is refused and with which words, that unusual but
allowed tensors reach the kernels with the right numbers, and the C interface's own refusals.

The tensors are fakes on "cuda:0": sizes, types and strides, no memory, so that nothing can be launched."""
from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
import warnings
from fractions import Fraction
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import min_fa3_op
from min_fa3_demo_b200 import _cabi, autograd, build, cache, min_fa3_op as op, rotary

warnings.filterwarnings("ignore", message="Accessing the data pointer of FakeTensor")
PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def test_root_module_exports():
    for name in ("RotaryAxes", "rotary", "append_cache", "forward_tree", "cache_weights", "evict_cache"):
        assert name in op.__all__ and getattr(min_fa3_op, name) is getattr(op, name)
    assert op.rotary is rotary.rotary and op.forward_tree is cache.forward_tree and autograd.rotary is not op.rotary


# ---------------------------------------------------------------------------------------
# Axes
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("freq", [0.0, 1.0, -1.0, 0.1, 1e-12, 5e-324, 123456.789, 2.0**80, 1e6 ** (-63 / 64)])
def test_turns_are_exact(freq):
    # In units of 2^-64 of a turn, to the nearest; a constant of 192 bits is exact for all but frequencies of 2^100.
    assert rotary._turn(freq) == round(Fraction(freq) * 2**64 / (2 * PI)) % 2**64


def test_axes_of_sections():
    a = rotary.RotaryAxes.from_sections((16, 24, 24), 1e6)
    assert (a.pairs, a.axes) == (64, 3) and list(a._c.axis) == [0] * 16 + [1] * 24 + [2] * 24
    assert list(a._c.turn) == [rotary._turn(1e6 ** (-i / 64)) for i in range(64)] and a._c.adjacent == 0
    b = rotary.RotaryAxes.from_sections((8, 0, 8), 1e4, restart=True, adjacent=True)
    assert (b.pairs, b.axes, b._c.adjacent) == (16, 3, 1)
    assert list(b._c.turn)[:16] == [rotary._turn(1e4 ** (-i / 8)) for i in range(8)] * 2


@pytest.mark.parametrize("make,words", [
    (lambda: rotary.RotaryAxes([1.0] * 7), "multiple of 8 between 8 and 64, got 7"),
    (lambda: rotary.RotaryAxes([1.0] * 72), "got 72"), (lambda: rotary.RotaryAxes([]), "got 0"),
    (lambda: rotary.RotaryAxes([1.0] * 8, [0] * 9), "same length. Got 8 vs 9"),
    (lambda: rotary.RotaryAxes([1.0] * 8, [0] * 7 + [-1]), "an axis must be between 0 and 63"),
    (lambda: rotary.RotaryAxes([float("inf")] * 8), "must be finite"),
    (lambda: rotary.RotaryAxes([float("nan")] * 8), "must be finite"),
    (lambda: rotary.RotaryAxes.from_sections((-8, 16)), "must not be negative"),
])
def test_axes_that_are_refused(make, words):
    with pytest.raises(RuntimeError, match=re.escape(words)):
        make()


# ---------------------------------------------------------------------------------------
# Calls
# ---------------------------------------------------------------------------------------
class Launched(Exception):
    pass


class Library:
    """Stands for the C library: keeps a call's arguments and goes no further."""

    STRUCTS = {"b2a_rotary": _cabi.RotaryArgs, "b2a_cache_append": _cabi.AppendArgs, "b2a_tree_fwd": _cabi.TreeArgs,
               "b2a_cache_weights": _cabi.TreeArgs, "b2a_cache_evict": _cabi.EvictArgs}

    def __getattr__(self, name):
        if name.endswith("_workspace_bytes"):
            return lambda *sizes: 1024

        def call(args, stream):
            raise Launched(self.STRUCTS[name].from_buffer_copy(args))
        return call


MODE = FakeTensorMode()


@pytest.fixture(params=["device known", "device new"])
def fake(request, monkeypatch):
    """Both ways through the checks: few expressions first, and, on a device not seen before, the list at once."""
    monkeypatch.setattr(op, "_SM100", {0} if request.param == "device known" else set())
    monkeypatch.setattr(cache, "_SM100", op._SM100)
    monkeypatch.setattr(rotary, "_SM100", op._SM100)
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda device=None: (10, 0))
    monkeypatch.setattr(_cabi, "load", lambda lib=Library(): lib)
    for module in (cache, rotary):
        monkeypatch.setattr(module, "_on_device", lambda device: op._HERE)
        monkeypatch.setattr(module, "_stream_ptr", lambda device: 0)
    with MODE:
        yield


def t(*shape, dtype=torch.bfloat16, device="cuda:0"):
    return torch.empty(shape, dtype=dtype, device=device)


def i32(*shape):
    return t(*shape, dtype=torch.int32)


AXES = rotary.RotaryAxes.from_sections((16, 24, 24))


def arguments(call):
    pages = dict(k_cache=t(9, 16, 2, 128), v_cache=t(9, 16, 2, 128), cache_lens=i32(3), block_table=i32(3, 4))
    if call == "rotary":
        return dict(q=t(3, 5, 4, 128), k=t(3, 5, 2, 128), positions=t(3, 3, 5, dtype=torch.int64), axes=AXES)
    if call == "append":
        return dict(k=t(3, 5, 2, 128), v=t(3, 5, 2, 128), **pages, q=t(3, 5, 4, 128), positions=i32(3, 3, 5), axes=AXES)
    if call == "append packed":
        return dict(k=t(11, 2, 128), v=t(11, 2, 128), **pages, cu_seqlens=i32(4), q=None, positions=None, axes=None)
    if call == "tree":
        return dict(q=t(3, 5, 4, 128), **pages, tree_mask=t(3, 5, 5, dtype=torch.bool), max_seqlen_q=None, cu_seqlens_q=None, out=None)
    if call == "tree packed":
        return dict(q=t(11, 4, 128), **pages, tree_mask=t(11, 6, dtype=torch.bool), max_seqlen_q=6, cu_seqlens_q=i32(4), out=None)
    if call == "weights":
        del pages["v_cache"]
        return dict(q=t(3, 5, 4, 128), lse=t(3, 4, 5, dtype=torch.float32), **pages, weights=t(3, 2, 64, dtype=torch.float32),
                    tree_mask=None, max_seqlen_q=5, cu_seqlens_q=None)
    return dict(**pages, weights=t(3, 2, 64, dtype=torch.float32), budget=40, recent=8)


FUNCTIONS = {"rotary": rotary.rotary, "append": cache.append_cache, "append packed": cache.append_cache, "tree": cache.forward_tree,
             "tree packed": cache.forward_tree, "weights": cache.cache_weights, "evict": cache.evict_cache}


def launch(call, **change):
    """The arguments that reach the library."""
    with pytest.raises(Launched) as caught:
        FUNCTIONS[call](**dict(arguments(call), **change))
    return caught.value.args[0]


@pytest.mark.parametrize("call", list(FUNCTIONS))
def test_calls_in_order_reach_the_library(fake, call):
    args = launch(call)
    if call == "rotary":
        assert (args.batch, args.seqlen, args.heads_q, args.heads_k, args.positions_64, args.inverse) == (3, 5, 4, 2, 1, 0)
        assert list(args.q_stride) == [2560, 512, 128] and list(args.positions_stride) == [15, 5, 1]
        return
    view = args.cache
    assert (view.pages, view.page_size, view.heads_k, view.table_width, view.table_stride) == (9, 16, 2, 4, 4)
    assert list(view.k_stride) == [4096, 256, 128] and args.batch == 3
    if call.startswith("tree"):
        assert (args.seqlen_q, args.total_q, args.heads_q) == ((5, 15, 4) if call == "tree" else (6, 11, 4))
        assert list(args.q_stride) == [512, 128] and list(args.mask_stride) == ([25, 5] if call == "tree" else [0, 6])
    if call == "weights":
        assert list(args.weights_stride) == [128, 64] and args.weights_slots == 64 and list(args.mask_stride) == [0, 0]
    if call == "append":
        assert (args.seqlen, args.total, args.heads_q, args.positions_64) == (5, 15, 4, 0)
    if call == "evict":
        assert (args.budget, args.recent, args.weights_slots) == (40, 8, 64)


def test_unusual_tensors_reach_the_library(fake):
    # One sequence, whose stride nobody looks at; one token; a cache without pages; dimensions of one with odd strides.
    whole = dict(block_table=None, k_cache=t(4, 33, 2, 128), v_cache=t(4, 33, 2, 128))
    args = launch("tree", **whole)
    assert (args.cache.pages, args.cache.page_size, args.cache.table_width) == (4, 33, 1) and not args.cache.block_table
    one = dict(q=t(1, 9, 4, 128)[:, :5], cache_lens=i32(1), block_table=i32(1, 4), tree_mask=t(1, 5, 7, dtype=torch.bool)[..., :5])
    args = launch("tree", **one)
    assert list(args.q_stride) == [512, 128] and list(args.mask_stride) == [35, 7]
    args = launch("tree", q=t(3, 9, 4, 128)[:, 3:4], tree_mask=t(3, 1, 1, dtype=torch.bool))
    assert list(args.q_stride) == [9 * 512, 128] and args.seqlen_q == 1
    odd = t(9 * 16 * 128 + 3)
    single = torch.as_strided(odd, (9, 16, 1, 128), (2048, 128, 1, 1))
    args = launch("tree", q=t(3, 5, 4, 128), k_cache=single, v_cache=single)
    assert list(args.cache.k_stride) == [2048, 128, 0]
    args = launch("rotary", k=None, q=t(3, 5, 7, 128)[:, :, 1:5], positions=t(3, 1, 5, dtype=torch.int32).expand(-1, 3, -1))
    assert args.heads_k == 0 and list(args.q_stride) == [5 * 7 * 128, 7 * 128, 128] and list(args.positions_stride) == [5, 0, 1]
    args = launch("evict", weights=t(3, 5, 2, 70, dtype=torch.float32)[:, 2, :, 3:64], recent=0, budget=1)
    assert list(args.weights_stride) == [700, 70] and args.weights_slots == 61


def test_nothing_is_launched_for_no_tokens(fake):
    none = rotary.rotary(t(3, 0, 4, 128), None, t(3, 3, 0, dtype=torch.int64), AXES)
    assert none[0].shape == (3, 0, 4, 128) and none[1] is None
    a = arguments("append")
    assert cache.append_cache(**dict(a, k=t(3, 0, 2, 128), v=t(3, 0, 2, 128), q=None, positions=None, axes=None)) is None
    a = arguments("tree packed")
    out, lse = cache.forward_tree(**dict(a, q=t(0, 4, 128), tree_mask=None), return_lse=True)
    assert out.shape == (0, 4, 128) and lse.shape == (4, 0)


F32 = torch.float32
REFUSALS = [
    ("rotary", dict(q=lambda: t(3, 5, 4, 128, device="cpu")), "q must be a CUDA tensor"),
    ("rotary", dict(q=lambda: t(3, 5, 4, 128, dtype=F32)), "q must have dtype torch.bfloat16"),
    ("rotary", dict(q=lambda: t(5, 128)), "q must have shape [B, S, H, D] or [total_tokens, H, D]"),
    ("rotary", dict(q=lambda: t(3, 5, 4, 64)), "q must have head_dim D=128"),
    ("rotary", dict(q=lambda: t(3, 5, 4, 256)[..., ::2]), "with adjacent values in a head"),
    ("rotary", dict(q=lambda: t(3, 5, 4, 132)[..., :128]), "other strides multiples of 8"),
    ("rotary", dict(q=lambda: t(3, 5, 0, 128)), "q must have heads"), ("rotary", dict(k=lambda: t(3, 5, 0, 128)), "k must have heads"),
    ("append", dict(q=lambda: t(3, 5, 0, 128)), "q must have heads"),
    ("rotary", dict(k=lambda: t(3, 6, 2, 128)), "q and k must have the same tokens"),
    ("rotary", dict(k=lambda: t(15, 2, 128)), "k must have shape [B, S, H, D]"),
    ("rotary", dict(k=lambda: t(3, 5, 2, 128, device="cuda:1")), "q and k must be on the same CUDA device"),
    ("rotary", dict(positions=lambda: t(2, 3, 5, dtype=torch.int64)), "positions must have shape [3, 3, 5]. Got [2, 3, 5]"),
    ("rotary", dict(positions=lambda: t(3, 3, 5, dtype=F32)), "torch.int32 or torch.int64"),
    ("rotary", dict(positions=lambda: t(3, 3, 5, dtype=torch.int64, device="cpu")), "positions must be on the same CUDA device"),
    ("rotary", dict(axes=lambda: None), "axes must be a RotaryAxes"),
    ("append", dict(k=lambda: t(3, 5, 3, 128), v=lambda: t(3, 5, 3, 128)), "same KV head count. Got 3 vs 2"),
    ("append", dict(v=lambda: t(3, 4, 2, 128)), "k and v must have the same shape"),
    ("append", dict(k=lambda: t(2, 5, 2, 128), v=lambda: t(2, 5, 2, 128)), "k must have the batch size of cache_lens. Got 2 vs 3"),
    ("append", dict(axes=lambda: None), "positions and axes go together"),
    ("append", dict(axes=lambda: None, positions=lambda: None), "q is turned by positions"),
    ("append", dict(q=lambda: t(3, 6, 4, 128)), "q and k must have the same tokens"),
    ("append", dict(positions=lambda: i32(1, 3, 5)), "positions must have shape [3, 3, 5]"),
    ("append packed", dict(cu_seqlens=lambda: i32(3)), "cu_seqlens must have shape [4]. Got [3]"),
    ("append packed", dict(cu_seqlens=lambda: t(4, dtype=torch.int64)), "cu_seqlens must have dtype torch.int32"),
    ("append packed", dict(k=lambda: t(1, 11, 2, 128)), "k must have shape [total_tokens, H, D]"),
    *[(call, change, words) for call in ("append", "tree", "weights", "evict") for change, words in [
        (dict(k_cache=lambda: t(9, 16, 2, 128, dtype=torch.float16)), "k_cache must have dtype torch.bfloat16"),
        (dict(k_cache=lambda: t(9, 16, 256)), "k_cache must have shape [pages, page_size, KVH, D]"),
        (dict(k_cache=lambda: t(9, 16, 2, 64)), "k_cache must have head_dim D=128"),
        (dict(k_cache=lambda: t(0, 16, 2, 128)), "k_cache must not be empty"),
        (dict(k_cache=lambda: t(9, 16, 2, 132)[..., :128]), "k_cache must be 16-byte aligned"),
        (dict(k_cache=lambda: t(1, 16, 2, 128).expand(9, -1, -1, -1)), "k_cache must not be expanded"),
        (dict(cache_lens=lambda: t(3, dtype=torch.int64)), "cache_lens must have dtype torch.int32"),
        (dict(cache_lens=lambda: i32(3, 1)), "cache_lens must have shape [B]"),
        (dict(cache_lens=lambda: i32(0)), "cache_lens must have shape [B]"),
        (dict(cache_lens=lambda: i32(6)[::2]), "cache_lens must be contiguous"),
        (dict(cache_lens=lambda: torch.empty(3, dtype=torch.int32)), "cache_lens must be a CUDA tensor"),
        (dict(block_table=lambda: i32(2, 4)), "block_table must have shape [3, width]. Got [2, 4]"),
        (dict(block_table=lambda: i32(3, 0)), "block_table must have shape [3, width]. Got [3, 0]"),
        (dict(block_table=lambda: i32(4, 3).T), "the rows of block_table must be contiguous"),
        (dict(block_table=lambda: t(3, 4, dtype=torch.int64)), "block_table must have dtype torch.int32"),
        (dict(block_table=lambda: None, k_cache=lambda: t(2, 16, 2, 128), v_cache=lambda: t(2, 16, 2, 128)),
         "a cache without block_table needs a row for each sequence. Got 2 for 3"),
        (dict(k_cache=lambda: t(9, 12, 2, 128), v_cache=lambda: t(9, 12, 2, 128)), "page_size must be a multiple of 8. Got 12"),
    ]],
    *[(call, dict(v_cache=lambda: t(9, 16, 3, 128)), "k_cache and v_cache must have the same shape") for call in ("append", "tree", "evict")],
    *[(call, dict(v_cache=lambda: t(9, 16, 2, 128, device="cuda:1")), "must be on the same CUDA device") for call in ("append", "tree", "evict")],
    *[(call, change, words) for call in ("tree", "weights") for change, words in [
        (dict(q=lambda: t(3, 5, 3, 128)), "qhead % kvhead == 0 for GQA/MQA. Got qhead=3, kvhead=2"),
        (dict(q=lambda: t(3, 5, 258, 128)), "at most 128 query heads may share a KV head"),
        (dict(q=lambda: t(15, 4, 128)), "q must have shape [B, S, H, D]"),
        (dict(q=lambda: t(3, 9, 4, 128)[:, :5]), "q must have its sequences one behind the other"),
        (dict(q=lambda: t(3, 5, 1, 128).expand(-1, -1, 4, -1)), "q must not be expanded"),
        (dict(max_seqlen_q=lambda: 4), "max_seqlen_q must be q.size(1). Got 4 vs 5"),
        (dict(tree_mask=lambda: t(3, 5, 6, dtype=torch.bool)), "tree_mask must have shape [3, 5, 5]"),
        (dict(tree_mask=lambda: t(3, 5, 5, dtype=torch.uint8)), "tree_mask must have dtype torch.bool"),
        (dict(tree_mask=lambda: t(3, 5, 10, dtype=torch.bool)[..., ::2]), "the rows of tree_mask must be contiguous"),
    ]],
    ("tree packed", dict(max_seqlen_q=lambda: None), "packed q needs a positive max_seqlen_q"),
    ("tree packed", dict(max_seqlen_q=lambda: 0), "packed q needs a positive max_seqlen_q"),
    ("tree packed", dict(max_seqlen_q=lambda: 7), "tree_mask must have shape [11, max_seqlen_q or more]"),
    ("tree packed", dict(tree_mask=lambda: t(10, 6, dtype=torch.bool)), "tree_mask must have shape [11, max_seqlen_q or more]"),
    ("tree packed", dict(cu_seqlens_q=lambda: i32(3)), "cu_seqlens_q must have shape [4]"),
    ("tree", dict(out=lambda: t(3, 5, 4, 128).transpose(1, 2)), "out must be contiguous"),
    ("weights", dict(lse=lambda: t(3, 5, 4, dtype=F32)), "lse must be a contiguous torch.float32 tensor of shape [3, 4, 5]"),
    *[(call, change, words) for call in ("weights", "evict") for change, words in [
        (dict(weights=lambda: t(3, 2, 64)), "weights must have dtype torch.float32"),
        (dict(weights=lambda: t(3, 3, 64, dtype=F32)), "weights must have shape [3, 2, slots]"),
        (dict(weights=lambda: t(3, 2, 0, dtype=F32)), "weights must have shape [3, 2, slots]"),
        (dict(weights=lambda: t(3, 2, 128, dtype=F32)[..., ::2]), "the rows of weights must be contiguous"),
    ]],
    ("weights", dict(weights=lambda: t(3, 1, 64, dtype=F32).expand(-1, 2, -1)), "weights must not be expanded"),
    ("evict", dict(budget=lambda: 0), "budget must be positive. Got 0"),
    ("evict", dict(recent=lambda: 41), "recent must be between 0 and the budget. Got 41"),
    ("evict", dict(recent=lambda: -1), "recent must be between 0 and the budget. Got -1"),
]


@pytest.mark.parametrize("call,change,words", REFUSALS, ids=[f"{c}-{w[:40]}-{n}" for n, (c, _, w) in enumerate(REFUSALS)])
def test_refusals(fake, call, change, words):
    given = arguments(call)
    given.update((name, make()) for name, make in change.items() if name in given)      # cache_weights has no v_cache
    with pytest.raises(RuntimeError, match=re.escape(words)):
        FUNCTIONS[call](**given)


def test_other_devices_are_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda device=None: (9, 0))
    for name in ("_SM100",):
        for module in (op, cache, rotary):
            monkeypatch.setattr(module, name, set())
    with MODE:
        for call in FUNCTIONS:
            with pytest.raises(RuntimeError, match="only supports Blackwell SM100. Current device capability is 9.0"):
                FUNCTIONS[call](**arguments(call))


# ---------------------------------------------------------------------------------------
# The C interface
# ---------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    build.build()
    return _cabi.load()


def test_layouts(tmp_path):
    """The ctypes structures, the struct.pack formats and the header say the same."""
    gcc = shutil.which("gcc") or shutil.which("cc")
    if gcc is None:
        pytest.skip("no C compiler")
    header = Path(build.PKG_DIR).parent / "include" / "b200attn.h"
    structs = {"b2a_rotary_axes": _cabi.RotaryAxes, "b2a_rotary_args": _cabi.RotaryArgs, "b2a_cache": _cabi.Cache,
               "b2a_append_args": _cabi.AppendArgs, "b2a_tree_args": _cabi.TreeArgs, "b2a_evict_args": _cabi.EvictArgs}
    lines = "".join(f'printf("{name} %zu", sizeof({name}));' + "".join(f'printf(" %zu", offsetof({name}, {field[0]}));' for field in mirror._fields_)
                    + 'printf("\\n");\n' for name, mirror in structs.items())
    src = tmp_path / "sizes.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{header}"\nint main(void) {{\n{lines}return 0;\n}}\n')
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", str(src), "-o", str(tmp_path / "sizes")], check=True)
    for line in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size, *offsets = line.split()
        mirror = structs[name]
        assert ctypes.sizeof(mirror) == int(size), name
        assert [getattr(mirror, field[0]).offset for field in mirror._fields_] == [int(o) for o in offsets], name
    for pack, mirror in ((_cabi.ROTARY, _cabi.RotaryArgs), (_cabi.APPEND, _cabi.AppendArgs), (_cabi.TREE, _cabi.TreeArgs),
                         (_cabi.EVICT, _cabi.EvictArgs)):
        assert pack.size == ctypes.sizeof(mirror)
        flat = []

        def leaves(value):
            for field in value._fields_:
                v = getattr(value, field[0])
                if isinstance(v, ctypes.Structure):
                    leaves(v)
                elif isinstance(v, ctypes.Array):
                    flat.extend(v)
                else:
                    flat.append(v or 0)
        leaves(mirror.from_buffer_copy(pack.pack(*range(1, len(pack.unpack(bytes(pack.size))) + 1))))
        assert flat == list(range(1, len(flat) + 1)), mirror.__name__


def view(**change):
    fields = dict(k=256, v=256, block_table=256, table_stride=4, k_stride=(4096, 256, 128), v_stride=(4096, 256, 128), pages=9,
                  page_size=16, heads_k=2, table_width=4)
    fields.update(change)
    return fields


def filled(struct, fields):
    args = struct()
    for name, value in fields.items():
        if isinstance(value, dict):
            setattr(args, name, filled(_cabi.Cache, value))
        elif isinstance(value, tuple):
            getattr(args, name)[:] = value
        else:
            setattr(args, name, value)
    return args


def c_arguments(name):
    tree = dict(cache=view(), cache_lens=256, q=256, out=256, lse=256, q_stride=(512, 128), batch=3, seqlen_q=5, total_q=15, heads_q=4,
                weights=256, weights_stride=(128, 64), weights_slots=64, workspace=256, workspace_bytes=1 << 30)
    if name == "b2a_rotary":
        axes = rotary.RotaryAxes.from_sections((16, 24, 24))
        return _cabi.RotaryArgs, dict(axes=axes._at, q=256, k=256, q_out=256, k_out=256, positions=256, q_stride=(2560, 512, 128),
                                      k_stride=(1280, 256, 128), positions_stride=(15, 5, 1), batch=3, seqlen=5, heads_q=4, heads_k=2), axes
    if name == "b2a_cache_append":
        return _cabi.AppendArgs, dict(cache=view(), cache_lens=256, k=256, v=256, k_stride=(1280, 256, 128), v_stride=(1280, 256, 128),
                                      batch=3, seqlen=5, total=15, workspace=256, workspace_bytes=16), None
    if name == "b2a_cache_evict":
        return _cabi.EvictArgs, dict(cache=view(), cache_lens=256, weights=256, weights_stride=(128, 64), batch=3, weights_slots=64, budget=40,
                                     recent=8, new_lens=256, new_weights=256, index=256, workspace=256, workspace_bytes=1 << 30), None
    return _cabi.TreeArgs, tree, None


C_REFUSALS = [
    ("b2a_rotary", dict(axes=0), "axes must not be NULL"), ("b2a_rotary", dict(positions=0), "positions must not be NULL"),
    ("b2a_rotary", dict(q=8), "q must be a 16-byte aligned device pointer"), ("b2a_rotary", dict(k=0), "k must be a 16-byte aligned"),
    ("b2a_rotary", dict(q_stride=(2560, 511, 128)), "strides of q must be multiples of 8"),
    ("b2a_rotary", dict(q_out=0), "q_out and k_out must not be NULL"), ("b2a_rotary", dict(k_out=8), "must be 16-byte aligned"),
    ("b2a_rotary", dict(seqlen=0), "batch and seqlen must be positive"), ("b2a_rotary", dict(batch=1 << 20, seqlen=1 << 20), "fewer than 2^31"),
    ("b2a_cache_append", dict(cache_lens=0), "cache_lens must not be NULL"), ("b2a_cache_append", dict(total=14), "total = batch * seqlen"),
    ("b2a_cache_append", dict(q=256, heads_q=4), "q is turned by positions, so it needs axes"),
    ("b2a_cache_append", dict(workspace=0), "workspace must be a 16-byte aligned"),
    ("b2a_tree_fwd", dict(out=0), "out must be a 16-byte aligned"), ("b2a_tree_fwd", dict(heads_q=3), "heads_q % heads_k must be 0"),
    ("b2a_tree_fwd", dict(heads_q=258), "at most 128 query heads may share a K/V head"),
    ("b2a_tree_fwd", dict(total_q=14), "total_q = batch * seqlen_q"), ("b2a_tree_fwd", dict(lse=0), "q, lse and cache_lens must not be NULL"),
    ("b2a_cache_weights", dict(weights=0), "weights must not be NULL"), ("b2a_cache_weights", dict(weights_slots=0), "weights must not be NULL or empty"),
    ("b2a_cache_evict", dict(budget=0), "budget must be >= 1"), ("b2a_cache_evict", dict(recent=41), "recent must be between 0 and the budget"),
    ("b2a_cache_evict", dict(index=0), "must not be NULL"), ("b2a_cache_evict", dict(batch=40000), "at most 65535 sequences"),
    *[(name, dict(cache=view(**change)), words) for name in ("b2a_cache_append", "b2a_tree_fwd", "b2a_cache_evict") for change, words in [
        (dict(k=0), "the cache's k and v must not be NULL"), (dict(v=8), "the cache must be 16-byte aligned"),
        (dict(k_stride=(4096, 256, 100)), "strides of the cache must be multiples of 8"), (dict(pages=0), "must be positive"),
        (dict(page_size=12), "page_size must be a multiple of 8, got 12"), (dict(table_width=0), "at least one column"),
        (dict(page_size=1 << 16, table_width=1 << 16), "fewer than 2^31 slots"),
        (dict(block_table=0, pages=2), "needs a page for each sequence, got 2 for"),
    ]],
]


@pytest.mark.parametrize("name,change,words", C_REFUSALS, ids=[f"{n}-{w[:30]}-{i}" for i, (n, _, w) in enumerate(C_REFUSALS)])
def test_refusals_of_the_c_interface(lib, name, change, words):
    struct, fields, keep = c_arguments(name)
    if name == "b2a_cache_evict" and "batch" in change:
        fields["cache"] = view(heads_k=2)
    args = filled(struct, dict(fields, **change))
    assert getattr(lib, name)(ctypes.byref(args), None) == _cabi.B2A_ERR_INVALID_ARGUMENT
    assert words in _cabi.last_error()
    del keep


@pytest.mark.parametrize("name", ["b2a_rotary", "b2a_cache_append", "b2a_tree_fwd", "b2a_cache_weights", "b2a_cache_evict"])
def test_null_arguments(lib, name):
    assert getattr(lib, name)(None, None) == _cabi.B2A_ERR_INVALID_ARGUMENT and "args must not be NULL" in _cabi.last_error()


def test_workspace_sizes(lib):
    assert lib.b2a_cache_weights_workspace_bytes() == cache._WEIGHTS_WORKSPACE
    assert lib.b2a_cache_evict_workspace_bytes(3, 2, 40, 64) >= 3 * 2 * 40 * 4 and lib.b2a_cache_evict_workspace_bytes(0, 2, 40, 64) == 0


def test_kernels_begin_by_waiting_and_promise_nothing_of_what_they_read():
    """All of them are launched early (launch_early): they wait before they touch global memory, and no pointer is read-only."""
    found = set()
    for path in sorted(build.CSRC_DIR.glob("*.cu*")):
        source = path.read_text()
        if path.name not in ("b2a_rotary.cu", "b2a_tree.cu", "b2a_tree_few.cu", "b2a_weights.cu", "b2a_evict.cu"):
            continue
        assert not re.search(r"__restrict__|__ldg\b|ld\.global\.nc|<<<", source), path.name
        for name, body in re.findall(r"__global__ void __launch_bounds__\([^)]*\)\s*(\w+)\([^{]*?\)\s*\{(.*?)\n\}", source, re.S):
            found.add(name)
            assert "let_next_kernel_start();\n    wait_for_previous_kernel();" in body, name
    assert found == {"rotary_tokens", "tree_attention", "tree_combine", "tree_attention_few", "tree_combine_few", "tree_weights", "evict_select",
                     "evict_fill", "evict_shift"}


def test_slot_of_a_page_without_a_division():
    """entry_of: the high half of slot * (2^32 / page_size, rounded up) is the quotient or one more, for all slots below 2^31."""
    import random
    rng = random.Random(0)
    for page in [8, 16, 24, 48, 56, 64, 104, 128, 160, 256, 1000, 4096, 65528, 1 << 20, (1 << 30) + 8]:
        per_page = (0xFFFFFFFF // page + 1) & 0xFFFFFFFF
        for slot in [0, 1, page - 1, page, page + 1, 2**31 - 1, *(rng.randrange(2**31) for _ in range(200)),
                     *(max(0, min(2**31 - 1, k * page + d)) for k in (1, 7, 2**31 // page) for d in (-1, 0, 1))]:
            at = (slot * per_page) >> 32
            row = slot - at * page
            if row < 0:
                at, row = at - 1, row + page
            assert (at, row) == divmod(slot, page)
