"""Refusals of masked attention that need no GPU (the C entry checks its arguments before any device call), and the
layout of the modifier struct against the header."""
import ctypes
import os
import re

import pytest
import torch

from npu_ai_b200 import _lib, kernels


def _call(mods=None, B=1, H=4, Hk=2, Sq=8, Skv=8, D=64, scale=0.125, variant=0, q=16, out=16, out_dtype=0):
    p = ctypes.c_void_p
    st = (Sq * H * D, H * D, D)
    ks = (Skv * Hk * D, Hk * D, D)
    m = ctypes.byref(mods) if mods is not None else None
    return _lib.call("npub200_attention_masked", p(q), *st, p(16), *ks, p(16), *ks, p(out), *st, out_dtype, B, H, Hk, Sq,
                     Skv, D, ctypes.c_float(scale), m, None, 0, variant, None)


@pytest.mark.parametrize("kw", [dict(B=0), dict(Sq=0), dict(Skv=0), dict(H=4, Hk=3), dict(Hk=0), dict(scale=0.0),
                                dict(scale=-1.0), dict(scale=float("nan")), dict(q=None), dict(out=None), dict(q=8),
                                dict(out_dtype=2)])
def test_bad_arguments(kw):
    with pytest.raises(ValueError):
        _call(**kw)


@pytest.mark.parametrize("kw", [dict(D=20), dict(D=264), dict(variant=-1), dict(variant=65), dict(B=70000)])
def test_unsupported_requests(kw):
    with pytest.raises(RuntimeError, match="-3"):
        _call(**kw)


@pytest.mark.parametrize("mods,kw", [
    (dict(prefix=3), {}),
    (dict(prefixes=16), {}),
    (dict(softcap=-1.0), {}),
    (dict(softcap=float("nan")), {}),
    (dict(softcap=float("inf")), {}),
    (dict(softcap=1e-31), {}),
    (dict(softcap=2e38), {}),
    ({}, dict(scale=float("inf"))),
    (dict(doc_offsets=16, docs=1), dict(Skv=9)),
    (dict(doc_offsets=16, docs=-1), {}),
    (dict(distance_bias=16, max_distance=-1), {}),
    (dict(mask=16, mask_dtype=5), {}),
    (dict(mask=16, mask_dtype=1, mask_sq=-8), {}),
])
def test_bad_modifiers(mods, kw):
    with pytest.raises(ValueError):
        _call(_lib.AttentionMods(**mods), **kw)


def test_workspace_size_checks_its_arguments():
    n = ctypes.c_size_t(0)
    with pytest.raises(ValueError):
        _lib.call("npub200_attention_masked_workspace_size", 1, 4, 3, 1, 1, 64, 0, ctypes.byref(n))
    with pytest.raises(ValueError):
        _lib.call("npub200_attention_masked_workspace_size", 1, 4, 2, 1, 1, 64, 0, None)


def test_host_tensors_are_refused():
    t = torch.zeros(1, 16, 80, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        kernels.attention(t, t, t, 2, causal=True)


def test_struct_matches_the_header(tmp_path):
    """Field order and the size of npub200_attention_mods as the host compiler lays it out."""
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = open(os.path.join(root, "include", "npu_b200.h")).read()
    body = re.search(r"typedef struct npub200_attention_mods \{(.*?)\} npub200_attention_mods;", src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n for line in body.split(";") for n in re.findall(r"(\w+)\s*(?=,|$)", line.strip())]
    fields = [n for n, _ in _lib.AttentionMods._fields_]
    assert [n for n in names if n in fields] == fields and len(names) == len(fields)
    c = tmp_path / "s.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "npu_b200.h"\nint main(void) {\n' + "".join(
        f'printf("%zu ", offsetof(npub200_attention_mods, {n}));\n' for n in fields)
        + 'printf("%zu", sizeof(npub200_attention_mods)); return 0; }\n')
    exe = tmp_path / "s"
    subprocess.run(["gcc", f"-I{root}/include", str(c), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(_lib.AttentionMods, n).offset for n in fields] + [ctypes.sizeof(_lib.AttentionMods)]


@pytest.mark.parametrize("softcap,scale", [(1e30, 1e-16), (1e30, 1e-9), (1e-30, 1e9), (1e-30, 2e8), (0.0, 3e38)])
def test_scales_that_leave_32_bits(softcap, scale):
    """scale / softcap and scale log2 e have to be normal f32 numbers: 0 would average every key, infinity gives NaN."""
    with pytest.raises(ValueError, match="scale"):
        _call(_lib.AttentionMods(softcap=softcap), scale=scale)


@pytest.mark.parametrize("softcap,scale", [(1e30, 1.2e-8), (1e-30, 5e7), (0.0, 2e38), (0.0, 1e-30)])
def test_scales_at_the_ends_of_the_range_pass_the_check(softcap, scale):
    """The next check, of the mask's type, is the one that refuses these calls."""
    with pytest.raises(ValueError, match="mask dtype"):
        _call(_lib.AttentionMods(softcap=softcap, mask=16, mask_dtype=5), scale=scale)
