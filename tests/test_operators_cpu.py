"""Host side of the training-step operators, without a GPU: the rotary table
against 64-bit arithmetic, configurations that are refused, scratch sizes, and
calls without a context."""
import ctypes as C
import math
import subprocess
import sys
from fractions import Fraction

import pytest

import bwpp


def frequencies(R, base=10000.0, scaling="none", factor=1.0, context=4096.0, low=1.0, high=32.0):
    if scaling == "base":
        base = base * factor ** (R / (R - 2))
    out = []
    for i in range(R // 2):
        f = base ** (-2.0 * i / R)
        if scaling == "linear":
            f = f / factor
        if scaling == "parts":
            keep = min(1.0, max(0.0, (context * f / (2 * math.pi) - low) / (high - low)))
            f = f * keep + f / factor * (1 - keep)
        out.append(f)
    return out


@pytest.mark.parametrize("R", [2, 4, 6, 64, 96, 128, 256])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("base", 8.0), ("parts", 16.0)])
def test_rope_table(R, scaling, factor):
    if scaling == "base" and R == 2:
        pytest.skip("refused: one pair does not depend on the base")
    t = bwpp.rope_table(R, scaling=scaling, factor=factor, context=4096.0, amplitude=1.25)
    assert t.pairs == R // 2 and t.amplitude == 1.25
    for f, turn in zip(frequencies(R, scaling=scaling, factor=factor), t.turns):
        # 2^-64 turns; a few 64-bit roundings (2^-53 each) of the frequency
        want = Fraction(f / (2 * math.pi)) % 1
        assert abs(Fraction(turn, 1 << 64) - want) <= Fraction(8, 1 << 53) * want + Fraction(1, 1 << 63)
    assert all(v == 0 for v in list(t.turns)[R // 2:])


@pytest.mark.parametrize("position", [1, 4097, 999983, 2**31 - 1])
def test_rope_table_angle_at_far_positions(position):
    """position * turns mod 2^64 is the angle: 2^31 positions keep 2^-21 rad."""
    t = bwpp.rope_table(128)
    for f, turn in zip(frequencies(128), t.turns):
        got = (position * turn % (1 << 64)) / 2.0**64 * 2 * math.pi
        assert abs(math.sin(got) - math.sin(position * f)) <= 8 * 2.0**-53 * position + 1e-12


@pytest.mark.parametrize("kw", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=258),
                                dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, base=float("inf")),
                                dict(rotary_dim=8, amplitude=0.0), dict(rotary_dim=8, amplitude=float("nan")),
                                dict(rotary_dim=8, scaling="linear", factor=0.0),
                                dict(rotary_dim=8, scaling="base", factor=-1.0),
                                dict(rotary_dim=2, scaling="base", factor=2.0),
                                dict(rotary_dim=8, scaling="parts", factor=2.0, context=0.0),
                                dict(rotary_dim=8, scaling="parts", factor=2.0, context=64.0, low=4.0, high=4.0)])
def test_rope_table_refusals(kw):
    with pytest.raises(bwpp.BwppError) as e:
        bwpp.rope_table(**kw)
    assert e.value.status == bwpp.ERR_ARG


@pytest.mark.parametrize("kw", [dict(rotary_dim=4, base=1e200, factor=1e200), dict(rotary_dim=64, base=1e300, factor=1e10),
                                dict(rotary_dim=4, base=1e-200, factor=1e-200)])
def test_rope_table_of_a_base_out_of_range(kw):
    """base * factor^(R / (R - 2)) overflows or vanishes: without an error all
    pairs but the first would stand still, or turn by any amount."""
    with pytest.raises(bwpp.BwppError) as e:
        bwpp.rope_table(scaling="base", **kw)
    assert e.value.status == bwpp.ERR_ARG


def test_rope_table_null_and_unknown_scaling():
    lib = bwpp.load()
    cfg = bwpp.RopeConfig(8, 4, 10000.0, 1.0, 0.0, 1.0, 32.0, 1.0)
    t = bwpp.RopeTable()
    assert lib.bwpp_cuda_rope_table(C.byref(t), C.byref(cfg)) == bwpp.ERR_ARG
    assert lib.bwpp_cuda_rope_table(None, C.byref(cfg)) == bwpp.ERR_ARG
    assert lib.bwpp_cuda_rope_table(C.byref(t), None) == bwpp.ERR_ARG


def test_calls_without_a_context_are_errors():
    lib = bwpp.load()
    assert lib.bwpp_cuda_xent_fwd_bf16(None, *[None] * 5, C.byref(bwpp.XentParams())) == bwpp.ERR_ARG
    assert lib.bwpp_cuda_xent_bwd_bf16(None, *[None] * 7, C.byref(bwpp.XentParams())) == bwpp.ERR_ARG
    for name in ("bf16", "f16", "f32"):
        assert getattr(lib, f"bwpp_cuda_rope_{name}")(None, *[None] * 5, C.byref(bwpp.RopeTable()),
                                                      C.byref(bwpp.RopeParams())) == bwpp.ERR_ARG
        assert getattr(lib, f"bwpp_cuda_junction_fwd_{name}")(None, *[None] * 7,
                                                              C.byref(bwpp.JunctionParams())) == bwpp.ERR_ARG
        assert getattr(lib, f"bwpp_cuda_junction_bwd_{name}")(None, *[None] * 12,
                                                              C.byref(bwpp.JunctionParams())) == bwpp.ERR_ARG
    assert lib.bwpp_cuda_junction_bwd_workspace_size(None, 4, 4, 0) == 0


def test_xent_workspace_size():
    assert bwpp.xent_workspace_size(0, 10, 10, 10, 10) == 0
    small = bwpp.xent_workspace_size(64, 1000, 64, 64, 1000)
    assert small > 0
    # the scratch is for a piece of the vocabulary, not for all of it
    T, V, D = 8192, 32000, 2048
    assert bwpp.xent_workspace_size(T, V, D, D, V, backward=1) < T * V * 4
    assert bwpp.xent_workspace_size(T, V, D, D, V) < T * V * 4


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("vocab_major", [0, 1])
@pytest.mark.parametrize("T,V,D", [(1, 1000, 64), (150, 1112, 136), (777, 4096, 1024)])
def test_xent_workspace_size_covers_odd_addresses(T, V, D, vocab_major, backward):
    """W at an address that is not 16-byte aligned is packed, whatever its pitch:
    one piece of it (all of these) is part of the size."""
    ldw = D if vocab_major else V
    size = bwpp.xent_workspace_size(T, V, D, D, ldw, vocab_major, backward, 1)
    assert size == bwpp.xent_workspace_size(T, V, D, D, ldw + 1, vocab_major, backward, 1)
    # what is kept besides: x, and the pairs and hits or dlogit
    rest = T * D * 2 + (T * V * 2 if backward else (V + 127) // 128 * T * 8 + T * 4)
    assert size >= rest + V * D * 2


@pytest.mark.parametrize("T,V,D", [(4, 4, 2**32 - 1), (4, 4, 2**31 - 511), (2**32 - 1, 4, 4), (2**32 - 1, 4, 2**32 - 1),
                                   (4, 2**32 - 1, 4), (4, 0, 4), (4, 4, 0)])
@pytest.mark.parametrize("vocab_major", [0, 1])
@pytest.mark.parametrize("backward", [0, 1])
def test_xent_workspace_size_of_sizes_that_are_refused(T, V, D, vocab_major, backward):
    """No scratch, and no arithmetic that wraps: a process of its own, as a
    division by a size that wrapped to zero ends it."""
    code = (f"import sys; sys.path[:0] = {sys.path!r}; import bwpp; "
            f"print(bwpp.xent_workspace_size({T}, {V}, {D}, {D}, {D if vocab_major else V}, {vocab_major}, {backward}))")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert (r.returncode, r.stdout.strip()) == (0, "0"), r


def test_struct_layouts():
    assert C.sizeof(bwpp.XentParams) == 40
    assert C.sizeof(bwpp.RopeTable) == 8 + 8 * bwpp.ROPE_MAX_PAIRS
    assert C.sizeof(bwpp.RopeParams) == 56
    assert C.sizeof(bwpp.JunctionParams) == 48


def test_packed_parameters_are_the_structs():
    xent = bwpp.XentParams.from_buffer_copy(bwpp._XENT.pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 0.5))
    assert [getattr(xent, n) for n, _ in xent._fields_] == [1, 2, 3, 4, 5, 6, 7, 8, 9, 0.5]
    rope = bwpp.RopeParams.from_buffer_copy(bwpp._ROPE.pack(*range(1, 10), -3, 11, 12, 13, 14))
    assert [getattr(rope, n) for n, _ in rope._fields_] == [*range(1, 10), -3, 11, 12, 13, 14]
    junction = bwpp.JunctionParams.from_buffer_copy(bwpp._JUNCTION.pack(*range(1, 9), 0.5, 1.5, 2.5, 3.5))
    assert [getattr(junction, n) for n, _ in junction._fields_] == [*range(1, 9), 0.5, 1.5, 2.5, 3.5]


def test_sizes_that_do_not_fit_their_field_are_errors():
    """2^32 rows would read as none."""
    with pytest.raises(Exception):
        bwpp._JUNCTION.pack(1 << 32, *range(7), 1.0, 1.0, 0.0, 0.0)
    with pytest.raises(Exception):
        bwpp._ROPE.pack(*range(9), 1 << 31, 0, 0, 0, 0)


@pytest.mark.parametrize("at", range(5))
@pytest.mark.parametrize("value", [1 << 32, (1 << 32) + 8, -1])
def test_workspace_sizes_that_do_not_fit_their_field_are_errors(at, value):
    sizes = [8] * 5
    sizes[at] = value
    with pytest.raises(Exception):
        bwpp.xent_workspace_size(*sizes)


@pytest.mark.parametrize("rotary_dim", [(1 << 32) + 8, -1])
def test_rotary_dims_that_do_not_fit_their_field_are_errors(rotary_dim):
    with pytest.raises(Exception):
        bwpp.rope_table(rotary_dim)


def test_packed_rope_config_is_the_struct():
    cfg = bwpp.RopeConfig.from_buffer_copy(bwpp._ROPE_CONFIG.pack(1, 2, 3.0, 4.0, 5.0, 6.0, 7.0, 8.5))
    assert [getattr(cfg, n) for n, _ in cfg._fields_] == [1, 2, 3.0, 4.0, 5.0, 6.0, 7.0, 8.5]
