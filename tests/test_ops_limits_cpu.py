"""radzero_amd.ops and the operators' C entries at the ends of what they take, without a GPU."""
import ctypes
import os
import subprocess
import sys

import pytest

from radzero_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("n_q", [5, 8])
def test_diff_attention_counts_the_workgroups_of_the_form_it_takes(lib, head_dim, n_q):
    """fp32 takes five to eight rows as two blocks: 2^23 sequences' key heads would be 2^24 workgroups of 256 threads, one more than a launch takes."""
    a = _lib.RzDiffAttentionArgs(dtype=0, batch=1 << 22, heads=2, kv_heads=2, n_q=n_q, n_k=5, head_dim=head_dim, causal=0, scale=0.125, lambda_init=0.2, out_scale=1.0, q_dev=16,
                                 k_dev=32, v_dev=48, out_dev=64, lambda_qk_dev=16)
    assert lib.rz_diff_attention(ctypes.byref(a), 16, 1 << 40, None) == 10001
    assert b"too many rows" in lib.rz_last_error()
    assert lib.rz_diff_attention_workspace(ctypes.byref(a)) == 0


@pytest.mark.parametrize("change", [lambda m: m.setitem(_lib.EXTRA_FLAGS, "rotary.hip", ["-g"]), lambda m: m.setitem(_lib.EXTRA_FLAGS, "diff_attention.hip", []),
                                    lambda m: m.setattr(_lib, "NO_PACKED_F32", []), lambda m: m.setattr(_lib, "ARCH", "gfx942"), lambda m: m.setattr(_lib, "LINK_FLAGS", []),
                                    lambda m: m.setenv("RZ_CXXFLAGS", "-DX=1"), lambda m: m.setattr(_lib, "SOURCES", _lib.SOURCES[1:])])
def test_every_flag_asks_for_a_new_library(monkeypatch, change):
    """A library built with other flags than the tree's is not taken for the tree's, and the same tree elsewhere asks for the same library."""
    was = _lib._source_digest()
    assert _lib._source_digest() == was and _lib.CSRC not in " ".join(_lib._flags())
    change(monkeypatch)
    assert _lib._source_digest() != was


def test_variants_are_compiled_as_the_library_is(tmp_path):
    """tools/build_variant.py leaves out none of the library's flags, the one against packed fp32 arithmetic among them."""
    _lib.build()                                         # current, so that the compiler below is asked for the variant alone
    said, compiler = tmp_path / "said", tmp_path / "hipcc"
    compiler.write_text(f'#!/bin/sh\necho "$@" >> {said}\n')
    compiler.chmod(0o755)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, os.path.join(root, "tools", "build_variant.py"), "x", "diff_attention.hip", "-DX=1"], check=True, env={**os.environ, "HIPCC": str(compiler)})
    compiled = said.read_text().splitlines()[0]
    for flag in [*_lib._flags(), *_lib.EXTRA_FLAGS["diff_attention.hip"], "-DX=1"]:
        assert flag in compiled.split(), flag
