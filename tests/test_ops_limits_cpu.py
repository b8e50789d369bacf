"""radzero_amd.ops and the operators' C entries at the ends of what they take, without a GPU."""
import ctypes
import os
import random
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


def places(p, n, stride, cols, size):
    """Addresses of the bytes of rows."""
    return {p + (i * stride[0] + j * stride[1] + k * stride[2] + c) * size + e for i in range(n[0]) for j in range(n[1]) for k in range(n[2]) for c in range(cols) for e in range(size)}


STRIDES = [0, 1, 3, 8, 16, 20, 24, 48, 50, 96, 100]


def test_rotary_refuses_outputs_that_overlap(lib):
    """Random strides and places against the sets of their bytes.  Positions are left out, so that the call ends there where nothing overlaps."""
    r, found = random.Random(7), [0, 0]
    for _ in range(4000):
        n, cols, dtype = (r.randint(1, 4), r.randint(1, 4), r.randint(1, 3)), r.choice([2, 4, 8]), r.choice([0, 1])
        strides = [[r.choice(STRIDES) for _ in n] for _ in range(2)]
        if r.random() < 0.4:
            strides[1] = strides[0]
        at = [4096 + 4 * r.randint(0, 300) for _ in range(2)]
        same = at[0] == at[1] and all(m == 1 or s == t for m, s, t in zip(n, *strides))
        want = not same and bool(places(at[0], n, strides[0], cols, 4 >> dtype) & places(at[1], n, strides[1], cols, 4 >> dtype))
        a = _lib.RzRotaryArgs(dtype=dtype, layout=0, batch=n[0], tokens=n[1], q_heads=n[2], k_heads=0, head_dim=cols, rotary_dim=2, n_axes=1, amplitude=1.0, q_dev=at[0], q_out_dev=at[1],
                              q_batch_stride=strides[0][0], q_token_stride=strides[0][1], q_head_stride=strides[0][2],
                              q_out_batch_stride=strides[1][0], q_out_token_stride=strides[1][1], q_out_head_stride=strides[1][2])
        assert lib.rz_rotary(ctypes.byref(a), None) == 10001
        assert (b"overlaps" in lib.rz_last_error()) == want, (n, cols, dtype, strides, at)
        found[want] += 1
    assert min(found) > 500


def test_rotary_refuses_outputs_whose_rows_overlap(lib):
    """Random strides, equal ones among them, against a count of the bytes."""
    r, found = random.Random(9), [0, 0]
    for _ in range(4000):
        n, cols, dtype = (r.randint(1, 4), r.randint(1, 4), r.randint(1, 3)), r.choice([2, 4, 8]), r.choice([0, 1])
        s = [r.choice(STRIDES) for _ in n]
        a = _lib.RzRotaryArgs(dtype=dtype, layout=0, batch=n[0], tokens=n[1], q_heads=n[2], k_heads=0, head_dim=cols, rotary_dim=2, n_axes=1, amplitude=1.0, q_dev=1 << 20, q_out_dev=4096,
                              q_batch_stride=1024, q_token_stride=128, q_head_stride=16, q_out_batch_stride=s[0], q_out_token_stride=s[1], q_out_head_stride=s[2])
        want = len(places(4096, n, s, cols, 4 >> dtype)) < n[0] * n[1] * n[2] * cols * (4 >> dtype)
        assert lib.rz_rotary(ctypes.byref(a), None) == 10001
        assert (b"rows overlap" in lib.rz_last_error()) == want, (n, cols, dtype, s)
        found[want] += 1
    assert min(found) > 500


def test_other_outputs_whose_rows_overlap(lib):
    a = _lib.RzDiffAttentionArgs(dtype=1, batch=1, heads=2, kv_heads=1, n_q=3, n_k=0, head_dim=32, scale=0.125, out_scale=1.0, q_dev=1 << 20, out_dev=4096, lambda_qk_dev=16,
                                 out_batch_stride=0, out_token_stride=64, out_head_stride=128)
    assert lib.rz_diff_attention(ctypes.byref(a), 16, 1 << 40, None) == 10001 and b"rows of out overlap" in lib.rz_last_error()
    for name in ("resid_out", "out"):
        a = _lib.RzResidualNormArgs(dtype=1, resid_dtype=0, batch=2, rows=3, dim=64, pre_kind=1, alpha=1.0, resid_dev=1 << 20, resid_batch_stride=192, resid_row_stride=64, scale_dev=16,
                                    **{name + "_dev": 4096, name + "_batch_stride": 128, name + "_row_stride": 64})
        assert lib.rz_residual_norm(ctypes.byref(a), None) == 10001 and b"rows overlap" in lib.rz_last_error()


def test_residual_norm_refuses_outputs_that_overlap(lib):
    """The same for x beside a residual of another type (a scale without y ends the call where nothing overlaps)."""
    r, found = random.Random(8), [0, 0]
    for _ in range(3000):
        n, cols, rt = (r.randint(1, 4), r.randint(1, 5), 1), r.choice([1, 3, 8]), r.choice([0, 1])
        strides = [[r.choice(STRIDES), r.choice(STRIDES), 0] for _ in range(2)]
        at = [4096 + 4 * r.randint(0, 200) for _ in range(2)]
        same = rt == 1 and at[0] == at[1] and all(m == 1 or s == t for m, s, t in zip(n, *strides))
        want = not same and bool(places(at[0], n, strides[0], cols, 4 >> rt) & places(at[1], n, strides[1], cols, 2))
        a = _lib.RzResidualNormArgs(dtype=1, resid_dtype=rt, batch=n[0], rows=n[1], dim=cols, pre_kind=1, alpha=1.0, resid_dev=at[0], out_dev=at[1], scale_dev=16,
                                    resid_batch_stride=strides[0][0], resid_row_stride=strides[0][1], out_batch_stride=strides[1][0], out_row_stride=strides[1][1])
        assert lib.rz_residual_norm(ctypes.byref(a), None) == 10001
        assert (b"overlaps" in lib.rz_last_error()) == want, (n, cols, rt, strides, at)
        found[want] += 1
    assert min(found) > 500


def test_overlaps_of_large_tensors(lib):
    """q, k and v of one projection, in place and crossed; a cache of 2^40 bytes; outputs that are each other."""
    b, n, h, d = 32, 5330, 12, 64
    at, step = 1 << 20, 36 * d
    heads = [at + 2 * i * h * d for i in range(3)]

    def rotary(q, k, qo, ko):
        layout = {f"{t}_{s}_stride": v for t in ("q", "k", "q_out", "k_out") for s, v in (("batch", n * step), ("token", step), ("head", d))}
        a = _lib.RzRotaryArgs(dtype=1, layout=0, batch=b, tokens=n, q_heads=h, k_heads=h, head_dim=d, rotary_dim=d, n_axes=1, amplitude=1.0, q_dev=q, k_dev=k, q_out_dev=qo, k_out_dev=ko, **layout)
        assert lib.rz_rotary(ctypes.byref(a), None) == 10001
        return b"overlaps" in lib.rz_last_error()

    q, k, v = heads
    far = at + 2 * b * n * step
    assert not rotary(q, k, q, k) and not rotary(q, q, far, far + 2 * h * d) and not rotary(q, k, v, far)
    assert rotary(q, k, k, q) and rotary(q, k, v, v) and rotary(q, k, q, q) and rotary(q, q, q, q) and rotary(q, k, q + 2 * d, far) and rotary(q, k, far, k - 2)

    a = _lib.RzDiffAttentionArgs(dtype=1, batch=4, heads=4, kv_heads=1, n_q=1, n_k=1 << 22, head_dim=64, scale=0.125, out_scale=1.0, q_dev=far, k_dev=at, v_dev=at + 256, lambda_qk_dev=16,
                                 q_batch_stride=512, q_token_stride=512, q_head_stride=128, out_batch_stride=512, out_token_stride=512, out_head_stride=128,
                                 k_batch_stride=1 << 37, k_token_stride=1 << 15, v_batch_stride=1 << 37, v_token_stride=1 << 15)
    for out in (at + 2 * 3 * (1 << 37) + 2 * (1 << 15) * ((1 << 22) - 1), at + 2 * (1 << 37) + 256 + 128, far + 1024):
        a.out_dev = out
        assert lib.rz_diff_attention(ctypes.byref(a), 16, 1 << 40, None) == 10001
        assert b"overlap" in lib.rz_last_error()

    a = _lib.RzResidualNormArgs(dtype=1, resid_dtype=1, batch=1, rows=1 << 30, dim=64, pre_kind=1, alpha=1.0, resid_dev=at, resid_out_dev=at, out_dev=at, scale_dev=16, resid_row_stride=64,
                                resid_out_row_stride=64, out_row_stride=64)
    assert lib.rz_residual_norm(ctypes.byref(a), None) == 10001 and b"outputs overlap" in lib.rz_last_error()
