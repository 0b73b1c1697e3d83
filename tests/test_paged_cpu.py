"""Rotary positions, the paged append and the paged attention without a GPU: what their C entries refuse before any device
call, the layout of their structs against the header, and the frequencies of each scaling."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

from npu_ai_b200 import _lib, kernels

P = ctypes.c_void_p
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rotation(freqs=16, rot_dim=64, magnitude=1.0, interleaved=0):
    return ctypes.byref(_lib.Rotation(freqs=freqs, rot_dim=rot_dim, magnitude=magnitude, interleaved=interleaved))


def cache(**kw):
    c = dict(k=16, k_sp=1024, k_ss=128, k_sh=64, v=16, v_sp=1024, v_ss=128, v_sh=64, pages=9, page_size=8, kv_heads=2,
             head_dim=64, table=16, table_stride=4, table_width=4)
    return _lib.PagedCache(**{**c, **kw})


def call_rope(x=16, st=(512, 256, 64), x_dtype=0, out=16, ost=(512, 256, 64), out_dtype=0, B=2, S=2, H=4, D=64, rot=None,
              start=0, starts=None, positions=None, pos=(0, 0), rot_none=False):
    _lib.call("npub200_rope", P(x), *st, x_dtype, P(out), *ost, out_dtype, B, S, H, D,
              None if rot_none else rot or rotation(), start, P(starts), P(positions), *pos, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(out=None), dict(x=17), dict(x_dtype=2), dict(out_dtype=7), dict(B=-1), dict(S=-1), dict(H=-1),
    dict(D=0), dict(st=(512, -256, 64)), dict(ost=(-8, 256, 64)), dict(rot_none=True), dict(rot=rotation(rot_dim=63)),
    dict(rot=rotation(rot_dim=66)), dict(rot=rotation(rot_dim=-2)), dict(rot=rotation(freqs=None)),
    dict(rot=rotation(freqs=12)), dict(rot=rotation(magnitude=math.nan)), dict(rot=rotation(magnitude=math.inf)),
    dict(starts=16, positions=16), dict(positions=16, pos=(-1, 1)), dict(start=2 ** 31), dict(start=-2 ** 31 - 1)])
def test_rope_bad_arguments(kw):
    with pytest.raises(ValueError):
        call_rope(**kw)


@pytest.mark.parametrize("kw", [dict(D=1026, rot=rotation()), dict(D=65), dict(H=65536), dict(B=2 ** 16, S=2 ** 15)])
def test_rope_unsupported(kw):
    with pytest.raises(RuntimeError, match="-3"):
        call_rope(**kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(S=0), dict(H=0)])
def test_rope_of_nothing_is_done(kw):
    call_rope(x=None, out=None, **kw)


def call_append(q=16, q_out=16, H=4, k=16, v=16, st=(512, 256, 64), dtype=0, c=None, starts=16, counts=None, B=2, S=2,
                rot=None, no_rot=False, no_cache=False):
    _lib.call("npub200_paged_append", P(q), *st, P(q_out), *st, H, P(k), *st, P(v), *st, dtype,
              None if no_cache else ctypes.byref(c or cache()), P(starts), P(counts), B, S,
              None if no_rot else rot or rotation(), None)


BAD_CACHES = [dict(k=None), dict(v=None), dict(k=17), dict(pages=-1), dict(page_size=0), dict(kv_heads=0), dict(head_dim=0),
              dict(table_width=-1), dict(table_stride=-4), dict(table=None), dict(k_sp=-1), dict(v_sh=-64)]


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(q_out=None), dict(k=None), dict(v=None), dict(starts=None), dict(dtype=2), dict(dtype=-1), dict(B=-1),
    dict(S=-2), dict(H=-1), dict(no_rot=True), dict(rot=rotation(rot_dim=80)), dict(no_cache=True), dict(q=17),
    dict(st=(512, 256, -64))] + [dict(c=cache(**c)) for c in BAD_CACHES])
def test_append_bad_arguments(kw):
    with pytest.raises(ValueError):
        call_append(**kw)


BIG_CACHES = [dict(page_size=2 ** 30, table_width=2), dict(page_size=1, table_width=2 ** 30 + 1), dict(pages=2 ** 31),
              dict(kv_heads=65536)]


@pytest.mark.parametrize("kw", [dict(c=cache(**c)) for c in BIG_CACHES] + [dict(c=cache(head_dim=66 * 16 + 2)), dict(H=70000)])
def test_append_unsupported(kw):
    with pytest.raises(RuntimeError, match="-3"):
        call_append(**kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(S=0)])
def test_append_of_nothing_is_done(kw):
    call_append(k=None, v=None, q=None, q_out=None, starts=None, **kw)


def call_attention(q=16, st=(512, 256, 64), c=None, lens=16, out=16, ost=(512, 256, 64), out_dtype=0, B=2, H=4, S=2,
                   scale=0.125, softcap=0.0, variant=0, no_cache=False):
    _lib.call("npub200_attention_paged", P(q), *st, None if no_cache else ctypes.byref(c or cache()), P(lens), P(out), *ost,
              out_dtype, B, H, S, ctypes.c_float(scale), 1, None, ctypes.c_float(softcap), None, None, 0, variant, None)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(out=None), dict(lens=None), dict(q=24), dict(out=17), dict(st=(512, 257, 64)), dict(st=(512, -256, 64)),
    dict(ost=(512, 256, -1)), dict(out_dtype=2), dict(B=-1), dict(S=-1), dict(H=0), dict(H=3), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(scale=3e38), dict(softcap=-1.0), dict(softcap=math.nan),
    dict(softcap=1e31), dict(softcap=1e-31), dict(softcap=1e30, scale=1e-9), dict(softcap=1e-30, scale=1e9),
    dict(no_cache=True), dict(c=cache(k=24)), dict(c=cache(v_ss=129)), dict(c=cache(k_sp=1028))]
    + [dict(c=cache(**c)) for c in BAD_CACHES])
def test_attention_bad_arguments(kw):
    with pytest.raises(ValueError):
        call_attention(**kw)


@pytest.mark.parametrize("kw", [dict(c=cache(**c)) for c in BIG_CACHES[:3]] + [
    dict(c=cache(head_dim=60)), dict(c=cache(head_dim=264)), dict(variant=-1), dict(variant=2 ** 20 + 1), dict(H=65536),
    dict(S=2 ** 25)])
def test_attention_unsupported(kw):
    with pytest.raises(RuntimeError, match="-3"):
        call_attention(**kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(S=0)])
def test_attention_of_nothing_is_done(kw):
    call_attention(q=None, out=None, lens=None, **kw)


@pytest.mark.parametrize("sizes", [(4, 3, 1, 64), (0, 1, 1, 64), (4, 2, 0, 64)])
def test_workspace_size_checks_its_arguments(sizes):
    n = ctypes.c_size_t(0)
    with pytest.raises(ValueError):
        _lib.call("npub200_attention_paged_workspace_size", *sizes, ctypes.byref(n))
    with pytest.raises(ValueError):
        _lib.call("npub200_attention_paged_workspace_size", 4, 2, 1, 64, None)


@pytest.mark.parametrize("name,struct", [("npub200_rotation", _lib.Rotation), ("npub200_paged_cache", _lib.PagedCache)])
def test_structs_match_the_header(tmp_path, name, struct):
    """Field order and sizes as the host compiler lays them out."""
    src = open(os.path.join(ROOT, "include", "npu_b200.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1), flags=re.S)
    names = [n for line in body.split(";") for n in re.findall(r"(\w+)\s*(?=,|$)", line.strip())]
    fields = [n for n, _ in struct._fields_]
    assert names == fields
    c = tmp_path / "s.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "npu_b200.h"\nint main(void) {\n' + "".join(
        f'printf("%zu ", offsetof({name}, {n}));\n' for n in fields) + f'printf("%zu", sizeof({name})); return 0; }}\n')
    exe = tmp_path / "s"
    subprocess.run(["gcc", f"-I{ROOT}/include", str(c), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(struct, n).offset for n in fields] + [ctypes.sizeof(struct)]


def test_host_tensors_are_refused():
    t = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    f = torch.zeros(32, dtype=torch.float64)
    pages = torch.zeros(4, 8, 2, 64, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        kernels.rope(t, f, 2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        kernels.paged_append(t, t, pages, pages, table, n)
    with pytest.raises(ValueError, match="CUDA tensor"):
        kernels.paged_attention(t, pages, pages, table, n, 2)
    with pytest.raises(NotImplementedError):
        _lib.torch_ops().rope(t, f, 2)


def test_frequencies():
    f, m = kernels.rope_frequencies(64, 500000.0)
    want = torch.tensor([500000.0 ** (-2 * j / 64) for j in range(32)], dtype=torch.float64)
    assert m == 1.0 and f.dtype == torch.float64 and torch.allclose(f, want, rtol=1e-14, atol=0.0)
    assert torch.equal(kernels.rope_frequencies(64, 500000.0, "linear", 4.0)[0], f / 4.0)
    ntk, m = kernels.rope_frequencies(64, 500000.0, "ntk", 8.0)
    assert m == 1.0 and ntk[0] == 1.0 and math.isclose(ntk[-1], f[-1] / 8.0, rel_tol=1e-12)
    yarn, m = kernels.rope_frequencies(64, 500000.0, "yarn", 16.0, original_length=8192)
    assert m == 0.1 * math.log(16.0) + 1.0
    for j in range(32):  # a pair's turns over the original length decide how much of its frequency stays
        turns = 8192 * float(f[j]) / (2 * math.pi)
        keep = min(1.0, max(0.0, math.log(turns) / math.log(32.0)))
        assert math.isclose(yarn[j], f[j] * keep + f[j] / 16.0 * (1.0 - keep), rel_tol=1e-12)
    assert kernels.rope_frequencies(2)[0].tolist() == [1.0]


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=7), dict(base=1.0), dict(factor=0.5), dict(scaling="other"),
                                dict(scaling="ntk", rot_dim=2), dict(beta_fast=1.0), dict(beta_slow=0.0),
                                dict(original_length=0), dict(base=math.nan)])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        kernels.rope_frequencies(**{"rot_dim": 64, **kw})


def test_tanh_of_the_cap_is_the_fitted_polynomial():
    """The cap's coefficients are those of the masked attention, which are fitted and checked by their own test."""
    csrc = os.path.join(ROOT, "npu_ai_b200", "csrc")
    found = [re.search(r"kTanhRatio\[6\] = \{(.*?)\}", open(os.path.join(csrc, f)).read(), re.S).group(1)
             for f in ("attention_masked.cuh", "attention_paged.cu")]
    a, b = ([float(x.rstrip("f")) for x in re.findall(r"-?\d[\d.e+-]*f", s)] for s in found)
    assert a == b and len(a) == 6


@pytest.mark.parametrize("d", list(range(1, 70)) + [127, 128, 129, 1000, 65535, 2 ** 20 + 1, 2 ** 30 - 1, 2 ** 30])
def test_division_by_multiplication(d):
    """csrc/fast_div.cuh: the same arithmetic on whole numbers, at the quotients' borders over its range."""
    log = max(0, (d - 1).bit_length())
    mul, shift = -(-2 ** (31 + log) // d), 31 + log
    assert mul < 2 ** 32
    for q in {0, 1, 2, (2 ** 31 - 1) // d // 2, (2 ** 31 - 1) // d}:
        for n in (q * d - 1, q * d, q * d + d - 1):
            if 0 <= n < 2 ** 31:
                assert (n * mul) >> shift == n // d


def test_schemas_name_what_is_written():
    """Tools that trust a schema would reorder or drop a call that says it writes nothing."""
    _lib.torch_ops()

    def written(name):
        schema = getattr(torch.ops.npub200, name).default._schema
        return schema.is_mutable, [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write]
    assert written("rope") == (True, ["out"])
    assert written("paged_append") == (True, ["k_pages", "v_pages", "q_out"])
    assert written("attention_paged") == (True, ["out"])


def test_whole_numbers_of_the_runner():
    """Numbers that int32 does not hold must not wrap to valid ones; types that hold no whole numbers are refused."""
    from npu_ai_b200.runner import _int32
    cpu = torch.device("cpu")
    low, high = -2 ** 31, 2 ** 31 - 1
    wide = torch.tensor([[-2 ** 63, 2 ** 32, 2 ** 32 + 5, -2 ** 32 + 3], [2 ** 63 - 1, low, high, 7]])
    assert _int32(wide, cpu, "t").tolist() == [[low, high, high, low], [high, low, high, 7]]
    assert _int32(torch.tensor([2 ** 32 - 1, 4], dtype=torch.uint32), cpu, "t").tolist() == [high, 4]
    for t in (torch.int8, torch.uint8, torch.int16, torch.uint16, torch.int32, torch.int64):
        for exact in (False, True):
            got = _int32(torch.tensor([0, 5, 127]).to(t), cpu, "t", exact)
            assert got.dtype == torch.int32 and got.tolist() == [0, 5, 127]
    assert _int32(torch.tensor([low, high]), cpu, "t", exact=True).tolist() == [low, high]
    for bad in (2 ** 31, low - 1, -2 ** 63):
        with pytest.raises(ValueError, match="32 bits"):
            _int32(torch.tensor([3, bad]), cpu, "t", exact=True)
    for t in (torch.float32, torch.float64, torch.bfloat16, torch.bool, torch.complex64, torch.uint64):
        with pytest.raises(ValueError, match="whole numbers"):
            _int32(torch.ones(2, dtype=t), cpu, "t")
    assert _int32(None, cpu, "t") is None and _int32(2 ** 40, cpu, "t", exact=True) == 2 ** 40


@pytest.fixture(scope="module")
def host_code(tmp_path_factory):
    """csrc/fast_div.cuh and csrc/paged_split.cuh as the host compiler builds them."""
    d = tmp_path_factory.mktemp("host")
    (d / "h.cpp").write_text(
        '#define __host__\n#define __device__\n#include "paged_split.cuh"\nusing namespace npub200;\n'
        'extern "C" int quotient(int64_t d, int n) { return divisor(d)(n); }\n'
        'extern "C" int64_t run(int64_t total, int blocks, int least, int workers) {\n'
        '  return tiles_of_run(total, blocks, divisor(blocks), least, workers);\n}\n')
    so = d / "h.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{ROOT}/npu_ai_b200/csrc",
                    str(d / "h.cpp"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.quotient.argtypes = [ctypes.c_int64, ctypes.c_int]
    lib.run.restype, lib.run.argtypes = ctypes.c_int64, [ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    return lib


def test_division_as_it_is_compiled(host_code):
    """Every quotient's borders over the divisors and the range that the kernels use."""
    for d in [*range(1, 70), 127, 128, 129, 296, 320, 1000, 65535, 2 ** 20 + 1, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1]:
        for q in {0, 1, 2, 3, (2 ** 31 - 1) // d // 2, (2 ** 31 - 1) // d - 1, (2 ** 31 - 1) // d}:
            for n in (q * d - 1, q * d, q * d + d // 2, q * d + d - 1):
                if 0 <= n < 2 ** 31:
                    assert host_code.quotient(d, n) == n // d, (d, n)


@pytest.mark.parametrize("blocks", [1, 148, 264, 296, 320])
@pytest.mark.parametrize("workers", [1, 2, 4])
def test_runs_are_the_least_that_hold_all_tiles(host_code, blocks, workers):
    for total in {*range(0, 40), *(k * blocks + e for k in (1, 2, 3, 4, 5, 8, 16, 31, 100, 2 ** 12) for e in (-1, 0, 1)),
                  *(2 ** 31 - blocks + e for e in (-1, 0, 1, 2)), 2 ** 20 - 1, 2 ** 20, 2 ** 31, 2 ** 40 + 3}:
        if total < 0:
            continue
        for least in (1, 3, 1000):
            run = host_code.run(total, blocks, least, workers)
            want = max(-(-total // blocks), least)
            assert run == -(-want // workers) * workers, (total, least)


def test_yarn_frequencies_between_whole_pairs():
    """The ramp from the 20th pair to the 46th (128 columns, base 10^4, 4096 tokens, turns of 32 and 1: the pairs 20.94 and
    45.03), and at ends that the head does not have."""
    f, _ = kernels.rope_frequencies(128)
    got, m = kernels.rope_frequencies(128, scaling="yarn", factor=16.0, whole_pairs=True)
    assert m == 0.1 * math.log(16.0) + 1.0
    for j in range(64):
        slow = min(1.0, max(0.0, (j - 20) / 26))
        assert math.isclose(got[j], float(f[j]) * (1.0 - slow) + float(f[j]) / 16.0 * slow, rel_tol=1e-12)
    plain = kernels.rope_frequencies(128, scaling="yarn", factor=16.0)[0]
    assert 0.3 < float((plain / got - 1.0).abs().max()) < 0.4  # what separates the two forms
    # 64 tokens: the pair of 32 turns lies before the first (-7.9), that of one turn at 16.1
    short = kernels.rope_frequencies(128, scaling="yarn", factor=4.0, original_length=64, whole_pairs=True)[0]
    for j in range(64):
        slow = min(1.0, j / 17)
        assert math.isclose(short[j], float(f[j]) * (1.0 - slow) + float(f[j]) / 4.0 * slow, rel_tol=1e-12)
    # a million tokens, 8 columns: the ramp would go from the 3rd pair, the head's last, to the 6th
    wide = kernels.rope_frequencies(8, scaling="yarn", factor=4.0, original_length=2 ** 20, whole_pairs=True)[0]
    assert wide.tolist() == kernels.rope_frequencies(8)[0].tolist()
    # both bounds behind the last column: nothing slows down; both before the first: everything from the second pair on
    assert torch.equal(kernels.rope_frequencies(8, 1.5, "yarn", 4.0, 2 ** 20, whole_pairs=True)[0],
                       kernels.rope_frequencies(8, 1.5)[0])
    tiny = kernels.rope_frequencies(8, scaling="yarn", factor=4.0, original_length=1, whole_pairs=True)[0]
    assert torch.allclose(tiny[1:], kernels.rope_frequencies(8)[0][1:] / 4.0, rtol=1e-12, atol=0.0) and tiny[0] == 1.0
    for scaling in (None, "linear", "ntk"):
        with pytest.raises(ValueError, match="whole_pairs"):
            kernels.rope_frequencies(64, scaling=scaling, whole_pairs=True)
