"""Arguments that the operators on int8 rows and beams refuse, through the C ABI and without a GPU: every check comes before
the context or the device is touched, so a block of zeros stands for the context."""
import ctypes as C

import numpy as np
import pytest

from needle_amd import _lib
from needle_amd.index import _state_layout

OK, ARG, UNSUPPORTED = _lib.OK, _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED
CTX = C.create_string_buffer(1 << 16)
MEM = np.zeros(1 << 20, dtype=np.uint8)  # pointers into it are never followed
BASE = (MEM.ctypes.data + 255) // 256 * 256


def at(offset):
    return BASE + offset


def quantize(ctx=CTX, rows=at(0), value=0, n=4, dim=8, row_stride=8, codes=at(4096), code_stride=8, scales=at(8192)):
    return _lib.lib().needle_hip_quantize_rows_i8_device(ctx, rows, value, n, dim, row_stride, codes, code_stride, scales)


@pytest.mark.parametrize("change,status", [
    (dict(ctx=None), ARG), (dict(value=3), ARG), (dict(value=-1), ARG), (dict(rows=None), ARG), (dict(codes=None), ARG), (dict(scales=None), ARG),
    (dict(row_stride=7), ARG), (dict(code_stride=7), ARG), (dict(rows=at(2)), ARG), (dict(value=1, rows=at(1)), ARG), (dict(scales=at(8193)), ARG),
    (dict(codes=at(100)), ARG), (dict(scales=at(4096 + 8)), ARG), (dict(scales=at(0)), ARG), (dict(row_stride=1 << 61), UNSUPPORTED),
    (dict(n=1 << 41), UNSUPPORTED), (dict(n=0), OK), (dict(n=0, rows=None, codes=None, scales=None), OK)])
def test_quantize_rows(change, status):
    assert quantize(**change) == status
    if status != OK:
        assert _lib.lib().needle_hip_last_error()


def product(linear=False, ctx=CTX, a=at(0), a_stride=64, a_scales=at(4096), m=4, b=at(8192), b_stride=64, b_scales=at(16384), n=8, k=64,
            bias=None, out_value=0, out=at(32768), out_stride=8, x_value=0):
    L = _lib.lib()
    if linear:
        return L.needle_hip_linear_i8_device(ctx, a, x_value, a_stride, m, b, b_stride, b_scales, n, k, bias, out_value, out, out_stride)
    return L.needle_hip_matmul_i8_device(ctx, a, a_stride, a_scales, m, b, b_stride, b_scales, n, k, bias, out_value, out, out_stride)


@pytest.mark.parametrize("linear", (False, True))
@pytest.mark.parametrize("change,status", [
    (dict(ctx=None), ARG), (dict(out_value=9), ARG), (dict(k=131072, a_stride=131072, b_stride=131072), UNSUPPORTED), (dict(n=1 << 31), UNSUPPORTED), (dict(m=1 << 31), UNSUPPORTED),
    (dict(a=None), ARG), (dict(b=None), ARG), (dict(b_scales=None), ARG), (dict(out=None), ARG), (dict(a_stride=63), ARG), (dict(b_stride=63), ARG),
    (dict(out_stride=7), ARG), (dict(out=at(32769)), ARG), (dict(bias=at(50001)), ARG), (dict(b_scales=at(16385)), ARG), (dict(out=at(0)), ARG),
    (dict(out=at(8192 + 64)), ARG), (dict(out=at(16384)), ARG), (dict(bias=at(32768)), ARG), (dict(out_stride=1 << 61), UNSUPPORTED),
    (dict(b_stride=1 << 62), UNSUPPORTED), (dict(m=0), OK), (dict(n=0), OK)])
def test_products(linear, change, status):
    assert product(linear, **change) == status


def test_products_in_their_own_way():
    assert product(a_scales=None) == ARG and product(a_scales=at(4097)) == ARG and product(out=at(4096)) == ARG
    assert product(True, x_value=5) == ARG and product(True, a=at(2)) == ARG


def select(ctx=CTX, logits=at(0), parents=at(1 << 18), tokens=at((1 << 18) + 4096), scores=at((1 << 18) + 8192), counts=at((1 << 18) + 12288),
           states=None, n_states=0, params=True, **p):
    q = dict(groups=2, beams=3, vocab=100, k=4, value=0, normalize=1, row_stride=100, scores=None, finished=None, mask=None, mask_stride=0,
             end_token=0, reserved=0)
    q.update(p)
    return _lib.lib().needle_hip_beam_select_device(ctx, C.byref(_lib.BeamParams(**q)) if params else None, logits, states, n_states, parents, tokens,
                                                    scores, counts)


@pytest.mark.parametrize("change,status", [
    (dict(ctx=None), ARG), (dict(params=False), ARG), (dict(value=4), ARG), (dict(reserved=1), ARG), (dict(k=257), UNSUPPORTED),
    (dict(beams=1025), UNSUPPORTED), (dict(beams=1, vocab=1 << 31, row_stride=1 << 31), UNSUPPORTED), (dict(beams=1024, vocab=1 << 22, row_stride=1 << 22), UNSUPPORTED),
    (dict(groups=1 << 30, beams=2), UNSUPPORTED), (dict(groups=1 << 30, k=2, beams=1), UNSUPPORTED), (dict(logits=None), ARG), (dict(parents=None), ARG),
    (dict(tokens=None), ARG), (dict(counts=None), ARG), (dict(row_stride=99), ARG), (dict(mask=at(4096 * 9), mask_stride=3), ARG),
    (dict(finished=at(4096 * 9), end_token=100), ARG), (dict(logits=at(2)), ARG), (dict(value=2, logits=at(1)), ARG), (dict(mask=at(4096 * 9 + 2)), ARG),
    (dict(counts=at(1 << 18)), ARG), (dict(parents=at(400)), ARG), (dict(row_stride=1 << 62), UNSUPPORTED), (dict(groups=0), OK),
    (dict(n_states=1), ARG), (dict(n_states=257, states=(_lib.BeamState * 257)()), UNSUPPORTED)])
def test_select(change, status):
    assert select(**change) == status


def state(**change):
    """groups 2, beams 3, k 4: six rows of two runs of 32 bytes become eight."""
    s = dict(src=at(1 << 16), dst=at(1 << 17), outer=1, inner=2, bytes=32, src_outer_stride=0, src_row_stride=100, src_inner_stride=40,
             dst_outer_stride=0, dst_row_stride=100, dst_inner_stride=40)
    s.update(change)
    return s


def reorder(*states, ctx=CTX, parents=at(0), groups=2, beams=3, k=4):
    arr = (_lib.BeamState * len(states))(*[_lib.BeamState(**s) for s in states])
    return _lib.lib().needle_hip_beam_reorder_device(ctx, parents, groups, beams, k, arr, len(states))


@pytest.mark.parametrize("states,status", [
    ([state(src=None)], ARG), ([state(dst=None)], ARG), ([state(dst_inner_stride=31)], ARG), ([state(dst_row_stride=71)], ARG),
    ([state(outer=3, dst_outer_stride=300)], ARG), ([state(dst_row_stride=0)], ARG), ([state(dst=at((1 << 16) + 200))], ARG),
    ([state(dst=at(1 << 16))], ARG), ([state(), state(src=at(1 << 15))], ARG), ([state(), state(src=at(1 << 17), dst=at(1 << 18))], ARG),
    ([state(dst_row_stride=1 << 61)], UNSUPPORTED), ([state(src_row_stride=1 << 61)], UNSUPPORTED), ([], OK),
    ([state(inner=0, src=None, dst=None)], None)])
def test_states(states, status):
    got = reorder(*states)
    assert got == status if status is not None else got in (_lib.ERR_HIP, _lib.OK)  # nothing to refuse: only the device is missing
    assert reorder(state(), ctx=None) == ARG and reorder(state(), parents=None) == ARG
    assert reorder(state(), groups=0) == OK and reorder(state(), k=0) == OK
    assert reorder(state(), parents=at((1 << 17) + 400)) == ARG
    for other in (dict(logits=at(1 << 17)), dict(parents=at(1 << 17)), dict(scores=at((1 << 17) + 100)), dict(counts=at((1 << 17) + 700)),
                  dict(finished=at(1 << 17)), dict(mask=at(1 << 17))):
        assert select(states=(_lib.BeamState * 1)(_lib.BeamState(**state())), n_states=1, **other) == ARG


def _bytes_of(s, side, rows):
    outer, row, inner = (s[f"{side}_{axis}_stride"] for axis in ("outer", "row", "inner"))
    return {s[side] + o * outer + r * row + i * inner + b for o in range(s["outer"]) for r in range(rows) for i in range(s["inner"]) for b in range(s["bytes"])}


def test_states_that_share_an_array_and_no_byte():
    """Keys and values as parts of every row, of every layer or of every run of one array lie between each other; a byte
    more and they overlap."""
    nothing_to_refuse = (_lib.ERR_HIP, OK)  # (only the device is missing)

    def pair(first, second):
        out = []
        for off in (first, second):
            out.append(dict(state(), src=at(1 << 16) + off, dst=at(1 << 17) + off))
        return out

    rows = dict(src_row_stride=160, dst_row_stride=160)  # six rows of two parts of 72 bytes (two runs of 32, 40 apart)
    apart = [[dict(s, **rows) for s in pair(0, 80)], [dict(s, **rows) for s in pair(88, 0)], [dict(s, **rows, outer=2, src_outer_stride=6 * 160, dst_outer_stride=8 * 160) for s in pair(0, 80)],
             pair(0, 0)[:1] + [dict(pair(0, 0)[1], src=at(1 << 16) + 32, dst=at(1 << 17) + 32, bytes=8)],  # in the gaps of the runs
             [dict(s, **rows, inner=4, bytes=20, src_inner_stride=40, dst_inner_stride=40) for s in pair(0, 20)]]
    for states in apart:
        assert reorder(*states) in nothing_to_refuse and reorder(*states[::-1]) in nothing_to_refuse
    meet = [[dict(s, **rows) for s in pair(0, 71)], [dict(s, **rows) for s in pair(0, 89)], [dict(s, **rows) for s in pair(0, 0)],
            pair(0, 0)[:1] + [dict(pair(0, 0)[1], src=at(1 << 16) + 32, dst=at(1 << 17) + 32, bytes=9)],
            [dict(s, **rows, inner=4, bytes=21, src_inner_stride=40, dst_inner_stride=40) for s in pair(0, 20)]]
    for states in meet:
        assert reorder(*states) == ARG and reorder(*states[::-1]) == ARG
    # a dst between the rows of a src
    assert reorder(state(dst=at((1 << 16) + 80), src_row_stride=160, dst_row_stride=160)) in nothing_to_refuse
    assert reorder(state(dst=at((1 << 16) + 71), src_row_stride=160, dst_row_stride=160)) == ARG
    rng = np.random.default_rng(0)
    taken = 0
    for _ in range(3000):  # whatever shares a byte is refused, whatever the strides
        stride = [int(v) for v in rng.choice([8, 12, 24, 48, 50, 96, 100, 200, 400], 6)]
        both = []
        for j in range(2):
            o, r, i = stride[:3] if rng.random() < 0.6 else stride[3:]
            both.append(dict(src=at(1 << 18) + j * (1 << 15), dst=at(1 << 17) + int(rng.integers(0, 120)), outer=int(rng.integers(1, 3)), inner=int(rng.integers(1, 4)),
                             bytes=int(rng.integers(1, 25)), src_outer_stride=8192, src_row_stride=1024, src_inner_stride=64, dst_outer_stride=o,
                             dst_row_stride=r, dst_inner_stride=i))
        if any(reorder(s) == ARG for s in both):  # (its own rows overlap)
            continue
        one, two = (_bytes_of(s, "dst", 8) for s in both)
        got = reorder(*both)
        if one & two:
            assert got == ARG, both
        elif max(one) < min(two) or max(two) < min(one):
            assert got in nothing_to_refuse, both
        taken += got in nothing_to_refuse
    assert taken > 20


def test_state_layouts():
    import torch

    src, dst = torch.zeros(6, 3, 20, 64, dtype=torch.bfloat16), torch.zeros(8, 3, 20, 64, dtype=torch.bfloat16)
    assert _state_layout(src, dst, 0) == (1, 1, 3 * 20 * 64 * 2, (0, 7680, 0), (0, 7680, 0))
    assert _state_layout(src[:, :, :5], dst[:, :, :5], 0) == (1, 3, 640, (0, 7680, 2560), (0, 7680, 2560))
    assert _state_layout(src[:, :1, :, 7:8], dst[:, :1, :, 7:8], 0) == (1, 20, 2, (0, 7680, 128), (0, 7680, 128))
    a, b = torch.zeros(2, 5, 6, 9), torch.zeros(2, 5, 8, 9)
    assert _state_layout(a, b, 2) == (10, 1, 36, (216, 36, 0), (288, 36, 0))
    with pytest.raises(ValueError):
        _state_layout(a[:, :2], b[:, :2], 2)  # two dimensions before the rows that do not fold
    with pytest.raises(ValueError):
        _state_layout(src[:, :2, :5, ::2], dst[:, :2, :5, ::2], 0)


def test_python_checks():
    """The object layer refuses before it calls the library."""
    import torch

    from needle_amd import Context

    c = Context.__new__(Context)
    c.device, c._h = 0, C.c_void_p()
    f, i8 = torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int8)
    s = torch.zeros(4)
    bad = [lambda: c.quantize_rows_device(f.double(), i8, s), lambda: c.quantize_rows_device(f, i8.int(), s), lambda: c.quantize_rows_device(f.T, i8, s),
           lambda: c.quantize_rows_device(f, i8, s[:3]), lambda: c.quantize_rows_device(f, i8, s), lambda: c.quantize_rows_device(f[0].expand(4, 8), i8, s),
           lambda: c.quantize_rows(np.zeros(4, np.float32)),
           lambda: c.matmul_i8_device(i8, s, i8[:, :4], s, torch.zeros(4, 4)), lambda: c.matmul_i8_device(i8, s, i8, s, torch.zeros(4, 5)),
           lambda: c.matmul_i8_device(f, s, i8, s, torch.zeros(4, 4)), lambda: c.matmul_i8_device(i8, s, i8, s, torch.zeros(4, 4)),
           lambda: c.matmul_i8_device(i8, s, i8, s, torch.zeros(4, 4, dtype=torch.int32)), lambda: c.linear_i8_device(i8, i8, s, torch.zeros(4, 4)),
           lambda: c.matmul_i8(np.zeros((4, 8)), np.zeros(4), np.zeros((4, 8), np.int8), np.zeros(4)),
           lambda: c.matmul_i8(np.zeros((4, 8), np.int8), np.zeros(3), np.zeros((4, 8), np.int8), np.zeros(4)),
           lambda: c.matmul_i8(np.zeros((4, 8), np.int8), np.zeros(4), np.zeros((4, 9), np.int8), np.zeros(4)),
           lambda: c.beam_select(np.zeros((4, 8)), None, 2, beams=3), lambda: c.beam_select(np.zeros((4, 8)), np.zeros(3), 2, beams=2),
           lambda: c.beam_select(np.zeros((4, 8)), None, 2, beams=2, mask=np.ones(7, bool))]
    i = torch.zeros(2, 3, dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)

    def sel(logits=f, scores=s, k=3, p=i, t=i, o=torch.zeros(2, 3), cnt=n, beams=2, **kw):
        return lambda: c.beam_select_device(logits, scores, k, p, t, o, cnt, beams=beams, **kw)

    bad += [sel(), sel(beams=3), sel(beams=0), sel(logits=f.double()), sel(scores=s[:2]), sel(p=i.long()), sel(cnt=torch.zeros(3, dtype=torch.int32)),
            sel(o=torch.zeros(2, 3).half()), sel(d_mask=torch.zeros(4, 2, dtype=torch.int32)), sel(d_mask=torch.zeros(2, 1, dtype=torch.int32)),
            sel(d_finished=torch.zeros(4)), sel(d_finished=torch.zeros(3, dtype=torch.bool)), sel(states=[(f, torch.zeros(6, 8))]),
            sel(states=[(f, torch.zeros(5, 8))]), sel(states=[(f, torch.zeros(6, 9))]), sel(states=[(f, torch.zeros(6, 8).half())])]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_python_passes_no_size_that_32_bits_cut():
    """Sizes and numbers the library takes in 32 bits are refused from 2^32 on, not cut to what is left of them: a row of 2^32 +
    16 codes is not one of 16."""
    import torch

    from needle_amd import Context

    c = Context.__new__(Context)
    c.device, c._h = 0, C.c_void_p()
    huge = (1 << 32) + 16

    def on(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="meta")  # a shape, and no memory

    def host(*shape, dtype=np.float32):
        return np.broadcast_to(np.zeros((), dtype), shape)

    i8, half = torch.int8, torch.float16
    i, n = on(1, 2, dtype=torch.int32), on(1, dtype=torch.int32)

    def sel(logits=on(1, 8), k=2, p=i, t=i, o=on(1, 2), cnt=n, beams=1, **kw):
        return lambda: c.beam_select_device(logits, None, k, p, t, o, cnt, beams=beams, **kw)

    wide = dict(p=on(1, huge, dtype=torch.int32), t=on(1, huge, dtype=torch.int32), o=on(1, huge))
    many = dict(p=on(huge, 1, dtype=torch.int32), t=on(huge, 1, dtype=torch.int32), o=on(huge, 1), cnt=on(huge, dtype=torch.int32))
    calls = [lambda: c.quantize_rows_device(on(1, huge, dtype=half), on(1, huge, dtype=i8), on(1)),
             lambda: c.quantize_rows(host(1, huge)), lambda: c.quantize_rows(host(1, huge, dtype=np.float16)),
             lambda: c.matmul_i8_device(on(1, huge, dtype=i8), on(1), on(2, huge, dtype=i8), on(2), on(1, 2)),
             lambda: c.matmul_i8_device(on(huge, 3, dtype=i8), on(huge), on(1, 3, dtype=i8), on(1), on(huge, 1)),
             lambda: c.linear_i8_device(on(1, huge), on(2, huge, dtype=i8), on(2), on(1, 2)),
             lambda: c.linear_i8_device(on(huge, 3), on(1, 3, dtype=i8), on(1), on(huge, 1)),
             lambda: c.matmul_i8(host(1, huge, dtype=np.int8), np.ones(1), host(2, huge, dtype=np.int8), np.ones(2)),
             lambda: c.matmul_i8(host(huge, 3, dtype=np.int8), host(huge), host(2, 3, dtype=np.int8), np.ones(2)),
             sel(logits=on(1, huge)), sel(k=huge, **wide), sel(logits=on(huge, 1), k=1, **many), sel(logits=on(0, 8), beams=huge, k=1, p=i[:0], t=i[:0], o=on(0, 1), cnt=n[:0]),
             lambda: c.beam_select(host(1, huge), None, 2, beams=1), lambda: c.beam_select(host(huge, 1), None, 2, beams=1),
             lambda: c.beam_select(host(1, 8), None, huge, beams=1),
             lambda: c.beam_reorder_device(on(1, 2, dtype=torch.int32), [(on(huge, 1, dtype=i8), on(2, 1, dtype=i8))], beams=huge),
             lambda: c.beam_reorder_device(on(1, huge, dtype=torch.int32), [(on(2, 1, dtype=i8), on(huge, 1, dtype=i8))], beams=2),
             lambda: c.beam_reorder_device(on(huge, 1, dtype=torch.int32), [(on(huge, 1, dtype=i8), on(huge, 1, dtype=i8))], beams=1)]
    for j, call in enumerate(calls):
        with pytest.raises(_lib.NeedleHipError) as e:
            call()
        assert e.value.status == UNSUPPORTED and str(huge) in str(e.value), j
    for end in (-1, huge, (1 << 32) + 3):  # an end token that is one of the vocabulary only in its lower 32 bits
        for call in (sel(d_finished=on(1, dtype=torch.bool), end_token=end), lambda: c.beam_select(np.zeros((1, 8)), None, 2, beams=1, finished=[0], end_token=end)):
            with pytest.raises(_lib.NeedleHipError) as e:
                call()
            assert e.value.status == ARG and str(end) in str(e.value)


def test_structs_and_constants_mirror_the_header():
    import os
    import re

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    header = open(os.path.join(root, "include", "needle_hip.h")).read()
    rust = open(os.path.join(root, "bindings", "rust", "needle-hip-sys", "src", "lib.rs")).read()

    def names(text, opener, pattern):
        body = text[text.index(opener):]
        body = re.sub(r"/\*.*?\*/|//[^\n]*", "", body[body.index("{") + 1: body.index("}")], flags=re.S)
        return re.findall(pattern, body)

    for struct, mirror in (("needle_beam_params", _lib.BeamParams), ("needle_beam_state", _lib.BeamState)):
        fields = [n for line in names(header, f"typedef struct {struct}", r"([^;]+);") for n in re.findall(r"([a-z_0-9]+)\s*(?:,|$)", line.strip())]
        assert [n for n, _ in mirror._fields_] == fields
        assert names(rust, f"pub struct {struct}", r"pub\s+([a-z_0-9]+)\s*:") == fields
    assert C.sizeof(_lib.BeamParams) == 72 and C.sizeof(_lib.BeamState) == 88
    for name, value in re.findall(r"\b(NEEDLE_VALUE_[A-Z0-9]+)\s*=\s*(\d+)", header):
        assert f"pub const {name}: c_int = {value};" in rust and getattr(_lib, name[len("NEEDLE_"):]) == int(value)


def test_build_rs_compiles_the_operators_as_the_makefile_does():
    import os
    import re

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    mk = open(os.path.join(root, "needle_amd", "csrc", "Makefile")).read()
    rs = open(os.path.join(root, "bindings", "rust", "needle-hip-sys", "build.rs")).read()
    objs = re.search(r"^OPERATOR_OBJS := (.*)$", mk, flags=re.M).group(1).split()
    flags = re.search(r"^OPERATOR_FLAGS := (.*)$", mk, flags=re.M).group(1).split()
    assert re.findall(r'"([^"]+)"', re.search(r"const OPERATOR_SOURCES[^=]*=([^;]*);", rs).group(1)) == [o.replace(".o", ".hip") for o in objs]
    assert re.findall(r'"([^"]+)"', re.search(r"const OPERATOR_FLAGS[^=]*=([^;]*);", rs).group(1)) == flags
