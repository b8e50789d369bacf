"""radzero_amd.ops without a GPU: what the operators refuse, before any kernel is launched, and the host-side frequency tables."""
import ctypes
import math

import pytest
import torch

from radzero_amd import _lib, ops


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_operators_have_no_cpu_fallback():
    q = torch.zeros(1, 2, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        ops.rotary(q, positions=torch.arange(2), freqs=torch.ones(32, dtype=torch.float64))
    with pytest.raises(ValueError, match="GPU"):
        ops.diff_attention(q, q, q, torch.zeros(4, 32), lambda_init=0.2)
    with pytest.raises(ValueError, match="GPU"):
        ops.residual_norm(q[0, 0], q[0, 0], pre_norm=ops.Norm())


def rotary_args(**kw):
    a = _lib.RzRotaryArgs(dtype=1, layout=0, batch=1, tokens=4, q_heads=2, k_heads=0, head_dim=64, rotary_dim=64, n_axes=1, amplitude=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [{"dtype": 3}, {"dtype": -1}, {"layout": 2}, {"batch": -1}, {"tokens": -1}, {"q_heads": 0}, {"k_heads": -1}, {"q_heads": 1 << 20}, {"rotary_dim": 63},
                                 {"rotary_dim": 66}, {"rotary_dim": 0}, {"head_dim": 1026}, {"n_axes": 0}, {"n_axes": 3}, {"tokens": 1 << 30, "batch": 4}, {}])
def test_rotary_refuses(lib, bad):
    assert lib.rz_rotary(ctypes.byref(rotary_args(**bad)), None) == 10001          # {}: null pointers
    assert b"rz_rotary" in lib.rz_last_error()


def test_rotary_of_nothing_is_no_work(lib):
    assert lib.rz_rotary(ctypes.byref(rotary_args(tokens=0)), None) == 0
    assert lib.rz_rotary(ctypes.byref(rotary_args(batch=0)), None) == 0
    assert lib.rz_rotary(None, None) == 10001


def attention_args(**kw):
    a = _lib.RzDiffAttentionArgs(dtype=1, batch=1, heads=4, kv_heads=2, n_q=3, n_k=5, head_dim=64, causal=0, scale=0.125, lambda_init=0.2, norm_eps=1e-5, out_scale=1.0,
                                 q_dev=16, k_dev=16, v_dev=16, out_dev=16, lambda_qk_dev=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [{"dtype": 3}, {"head_dim": 48}, {"head_dim": 0}, {"batch": -1}, {"n_q": -1}, {"n_k": -1}, {"heads": 0}, {"kv_heads": 0}, {"kv_heads": 3}, {"causal": 3},
                                 {"causal": -1}, {"scale": 0.0}, {"scale": -1.0}, {"scale": math.nan}, {"scale": math.inf}, {"norm_weight_dev": 16, "norm_eps": -1.0},
                                 {"norm_weight_dev": 16, "norm_eps": math.nan}, {"n_k": (1 << 30) + 1}, {"n_q": 1 << 30}, {"batch": 1 << 20, "n_q": 1 << 10},
                                 {"q_dev": None}, {"k_dev": None}, {"v_dev": None}, {"out_dev": None}, {"lambda_qk_dev": None}, {"q_dev": 8}, {"out_dev": 24},
                                 {"q_token_stride": 4}, {"k_head_stride": 12}, {"v_batch_stride": 2}, {"out_token_stride": 7}])
def test_diff_attention_refuses(lib, bad):
    a = attention_args(**bad)
    assert lib.rz_diff_attention(ctypes.byref(a), 16, 1 << 40, None) == 10001
    assert b"rz_diff_attention" in lib.rz_last_error()


def test_diff_attention_workspace_of_any_sizes(lib):
    """No keys, one key, one block too few or too many: the plan of the work comes out, and what it stores stays within what fills the chip once."""
    for dtype in (0, 1):
        for head_dim in (32, 64, 128):
            for n_q in (1, 2, 3, 5, 33, 200, 5000):
                for n_k in (0, 1, 63, 64, 65, 1000, 1 << 16, 1 << 30):
                    for batch, lens in ((1, None), (3, 16), (64, 16), (65, 16), (700, None)):
                        for causal in (0, 2):
                            a = attention_args(dtype=dtype, head_dim=head_dim, n_q=n_q, n_k=n_k, batch=batch, kv_lens_dev=lens, causal=causal)
                            assert lib.rz_diff_attention_workspace(ctypes.byref(a)) <= 2048 * 128 * (4 * head_dim + 4) * 4


def test_diff_attention_workspace_and_nothing_to_do(lib):
    assert lib.rz_diff_attention(None, None, 0, None) == 10001
    assert lib.rz_diff_attention(ctypes.byref(attention_args(n_q=0)), None, 0, None) == 0
    assert lib.rz_diff_attention(ctypes.byref(attention_args(batch=0)), None, 0, None) == 0
    assert lib.rz_diff_attention_workspace(ctypes.byref(attention_args(head_dim=48))) == 0
    for a in (attention_args(n_q=1, n_k=1 << 16), attention_args(n_q=1, n_k=1 << 20, dtype=0, head_dim=128), attention_args(n_q=193, n_k=11882)):
        need = lib.rz_diff_attention_workspace(ctypes.byref(a))
        if need:
            assert lib.rz_diff_attention(ctypes.byref(a), None, 0, None) == 10002          # no workspace, and one byte short of it
            assert lib.rz_diff_attention(ctypes.byref(a), 16, need - 1, None) == 10002
            assert lib.rz_diff_attention(ctypes.byref(a), 8, need, None) == 10001


@pytest.mark.parametrize("many", [{"batch": 1 << 23, "n_q": 1}, {"batch": 1 << 14, "n_q": 1 << 14, "heads": 4, "kv_heads": 4}])
def test_diff_attention_refuses_more_workgroups_than_a_launch_takes(lib, many):
    a = attention_args(**many)
    assert lib.rz_diff_attention_workspace(ctypes.byref(a)) == 0
    assert lib.rz_diff_attention(ctypes.byref(a), 16, 1 << 40, None) == 10001


@pytest.mark.parametrize("same", ["q_dev", "k_dev", "v_dev"])
def test_diff_attention_does_not_write_over_its_inputs(lib, same):
    a = attention_args(**{**dict(q_dev=1 << 12, k_dev=1 << 13, v_dev=1 << 14), same: 16})
    assert lib.rz_diff_attention(ctypes.byref(a), 16, 1 << 40, None) == 10001
    assert b"out must not be" in lib.rz_last_error()


def norm_args(**kw):
    a = _lib.RzResidualNormArgs(dtype=1, resid_dtype=0, batch=1, rows=3, dim=768, post_kind=0, pre_kind=1, alpha=1.0, post_eps=0.0, pre_eps=1e-6,
                                y_dev=16, resid_dev=16, resid_out_dev=16, out_dev=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [{"dtype": 3}, {"resid_dtype": 2}, {"batch": -1}, {"rows": -1}, {"dim": 0}, {"dim": 16385}, {"post_kind": 3}, {"pre_kind": -1}, {"pre_eps": -1.0},
                                 {"post_eps": math.nan}, {"resid_dev": None}, {"resid_out_dev": None, "out_dev": None}, {"y_dev": None, "post_kind": 1},
                                 {"y_dev": None, "scale_dev": 16}, {"y_dev": None, "gate_dev": 16}, {"batch": 1 << 16, "rows": 1 << 16}])
def test_residual_norm_refuses(lib, bad):
    assert lib.rz_residual_norm(ctypes.byref(norm_args(**bad)), None) == 10001
    assert b"rz_residual_norm" in lib.rz_last_error()


def test_residual_norm_of_nothing_is_no_work(lib):
    assert lib.rz_residual_norm(None, None) == 10001
    assert lib.rz_residual_norm(ctypes.byref(norm_args(rows=0)), None) == 0


def test_structs_have_the_size_the_compiler_gives_them(tmp_path):
    """The ctypes mirrors against the header itself (a field left out would shift every later one)."""
    import os
    import shutil
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    pairs = [("rz_rotary_args", _lib.RzRotaryArgs), ("rz_diff_attention_args", _lib.RzDiffAttentionArgs), ("rz_residual_norm_args", _lib.RzResidualNormArgs)]
    lines = [f'printf("%zu\\n", sizeof({c}));' for c, _ in pairs] + [f'printf("%zu\\n", offsetof({c}, {n}));' for c, t in pairs for n, _ in t._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "radzero_hip.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run([cc, "-I", inc, str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(t) for _, t in pairs] + [getattr(t, n).offset for _, t in pairs for n, _ in t._fields_]


def test_packed_structs_are_the_ctypes_ones():
    for t in (_lib.RzRotaryArgs, _lib.RzDiffAttentionArgs, _lib.RzResidualNormArgs):
        a, values = t(), []
        for i, (n, c) in enumerate(t._fields_):
            values.append(i + 0.5 if c is ctypes.c_float else i + 1)
            setattr(a, n, values[-1])
        packed = t.pack(*values)
        assert packed == bytes(a)[:len(packed)] and not any(bytes(a)[len(packed):])
        assert (ctypes.c_char * len(packed)).from_buffer_copy(packed).raw == packed


def test_rotary_frequencies():
    f, a = ops.rotary_frequencies(8, base=100.0)
    assert f.dtype == torch.float64 and a == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    f2, _ = ops.rotary_frequencies(8, axes=2, base=100.0)
    assert f2.shape == (2, 2) and torch.allclose(f2, torch.tensor([[1.0, 0.1], [1.0, 0.1]], dtype=torch.float64), rtol=1e-15)
    lin, a = ops.rotary_frequencies(8, base=100.0, scaling={"kind": "linear", "factor": 4})
    assert torch.allclose(lin, f / 4) and a == 1.0
    ntk, a = ops.rotary_frequencies(8, base=100.0, scaling={"kind": "ntk", "factor": 4})
    assert a == 1.0 and abs(float(ntk[0]) - 1.0) < 1e-15 and abs(float(ntk[-1] / f[-1]) - 0.25) < 1e-12
    yarn, a = ops.rotary_frequencies(128, scaling={"kind": "yarn", "factor": 8, "original_length": 4096})
    plain, _ = ops.rotary_frequencies(128)
    turns = plain * 4096 / (2 * math.pi)
    assert abs(a - (0.1 * math.log(8) + 1)) < 1e-15
    assert torch.equal(yarn[turns >= 32], plain[turns >= 32]) and torch.allclose(yarn[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    assert bool((yarn[1:] < yarn[:-1]).all())
    assert torch.equal(ops.rotary_frequencies(64, scaling={"kind": "yarn", "factor": 1, "original_length": 4096})[0], ops.rotary_frequencies(64)[0])
    for bad in ({"rotary_dim": 7}, {"rotary_dim": 8, "axes": 3}, {"rotary_dim": 8, "scaling": {"kind": "cubic", "factor": 2}}, {"rotary_dim": 8, "scaling": {"kind": "linear"}},
                {"rotary_dim": 8, "scaling": {"kind": "yarn", "factor": 2}}, {"rotary_dim": 2, "scaling": {"kind": "ntk", "factor": 2}}):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)
