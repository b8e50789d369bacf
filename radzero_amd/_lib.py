"""Build + load libradzero_hip.so (the C-ABI of include/radzero_hip.h) through ctypes.

There is NO fallback: if the library is missing or fails to load, importing the product path raises.
"""
from __future__ import annotations

import ctypes
import os
import struct
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
EXP_SRC = os.path.join(PKG_DIR, "..", "tools", "experiments")     # retired experiments' sources: tools build only, never product
# RZ_EXPERIMENTS=1: the TOOLS build (-DRZ_EXPERIMENTS: in-kernel stamp builds of gemm7 / gemm8, the retired attention shapes of rounds 1-2),
# its own library and object directory; the product and every test use the plain build.
EXPERIMENTS = os.environ.get("RZ_EXPERIMENTS") == "1"
LIB_PATH = os.environ.get("RZ_LIB_PATH") or os.path.join(PKG_DIR, "libradzero_hip_experiments.so" if EXPERIMENTS else "libradzero_hip.so")   # RZ_LIB_PATH: A/B of two builds in one gpurun call
SOURCES = ["gemm.hip", "gemm7.hip", "gemm8.hip", "attention.hip", "rowops.hip", "vlcabs.hip", "preprocess.hip", "rotary.hip", "diff_attention.hip", "residual_norm.hip", "api.hip"]
if EXPERIMENTS:
    # retired GEMM experiments, never faster than gemm8 inside the step: gemm10 / gemm11 (round 3: other K loops), gemm12 (round 4: two
    # 256x128 workgroups per CU so that epilogues overlap K loops; profiles/r04/gemm12_*.log).  They live in tools/experiments/ (with the
    # generated loops attention.hip's and gemm10.hip's experiment branches include) and are found through -I
    SOURCES += ["gemm10.hip", "gemm11.hip", "gemm12.hip"]
# attention.hip: fmaxf chains on MFMA outputs fuse into v_max3_f32 without a canonicalising v_max each
EXTRA_FLAGS = {"attention.hip": ["-fno-honor-nans"],
               # results of matrix instructions in ordinary registers wherever they fit: the fp32 kernels' vector instructions work on them, and every one in an
               # accumulation register costs a move each way (one block of 32 keys of head dim 64: 573 -> 421 vector instructions)
               "diff_attention.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"]}
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
# no packed fp32 arithmetic (v_pk_add_f32 / v_pk_mul_f32 / v_pk_fma_f32): hipcc -O3 makes it from ordinary float code, and on these machines some of its
# forms have given wrong results now and then, without an error.  (hipcc's host pass warns that it does not know the feature: harmless.)
NO_PACKED_F32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
LINK_FLAGS = [f"--offload-arch={ARCH}", "-shared", "-fPIC"]


def _flags() -> list:
    """What every source is compiled with, but for its include folders."""
    return [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function", "-Werror=uninitialized", "-Werror=return-type", *NO_PACKED_F32,
            *(["-DRZ_EXPERIMENTS"] if EXPERIMENTS else []), *os.environ.get("RZ_CXXFLAGS", "").split()]      # RZ_CXXFLAGS: A/B builds of a tunable (with RZ_LIB_PATH)

RZ_F32, RZ_BF16, RZ_F16 = 0, 1, 2
PROF_FAMILIES = ("attn", "gemm", "rowops", "vlcabs", "post")


def _src_path(src: str) -> str:
    p = os.path.join(CSRC, src)
    return p if os.path.exists(p) or not EXPERIMENTS else os.path.join(EXP_SRC, src)


def _all_deps() -> list:
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(PKG_DIR, "..", "include", "radzero_hip.h")]
    if EXPERIMENTS and os.path.isdir(EXP_SRC):
        deps += [os.path.join(EXP_SRC, f) for f in os.listdir(EXP_SRC)]
    return deps


STAMP_PATH = LIB_PATH + ".stamp"


def _source_digest() -> str:
    """sha256 over the CONTENTS of every source / header the library is built from (+ the sources' list and all flags): the rebuild decision must not
    depend on file times — a snapshot copied to another machine (gpurun, the driver's round-end run) keeps contents, not necessarily mtime order."""
    import hashlib
    h = hashlib.sha256()
    h.update(repr((SOURCES, _flags(), sorted(EXTRA_FLAGS.items()), LINK_FLAGS)).encode())
    for d in sorted(os.path.abspath(p) for p in _all_deps() if os.path.isfile(p)):
        h.update(os.path.basename(d).encode())
        with open(d, "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def _needs_rebuild() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    try:
        return open(STAMP_PATH).read().strip() != _source_digest()
    except OSError:
        pass
    # a library without a stamp (built by an older tree): fall back to file times
    t = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(d) > t for d in _all_deps() if os.path.exists(d))


def build(force: bool = False, verbose: bool = False) -> str:
    """hipcc --offload-arch=gfx950 every source, link in-tree (the .so travels with the repo snapshot).

    Safe under `torch.distributed.run` (every rank imports this module at the same time): the whole build runs under an
    exclusive `flock` on radzero_amd/build/.lock, objects and the library are written to per-process temporary names and
    moved into place with `os.replace`, and whoever gets the lock second finds an up-to-date library and does nothing.
    A reader therefore never maps a half-written file."""
    if not force and not _needs_rebuild():
        return LIB_PATH
    if not os.path.exists(HIPCC):
        raise RuntimeError(f"hipcc not found at {HIPCC}; cannot build libradzero_hip.so")
    import fcntl
    obj_dir = os.path.join(PKG_DIR, "build_experiments" if EXPERIMENTS else "build")
    if os.environ.get("RZ_CXXFLAGS", "").strip():        # an A/B build: its objects must never be mistaken for the product's (they are reused by file time alone)
        import hashlib
        obj_dir += "_" + hashlib.sha256(os.environ["RZ_CXXFLAGS"].encode()).hexdigest()[:10]
    os.makedirs(obj_dir, exist_ok=True)
    with open(os.path.join(obj_dir, ".lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            if not force and not _needs_rebuild():       # another process built it while this one waited
                return LIB_PATH
            return _build_locked(obj_dir, verbose, force)
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)


def _build_locked(obj_dir: str, verbose: bool, force: bool = False) -> str:
    flags = [*_flags(), f"-I{CSRC}", *([f"-I{EXP_SRC}"] if EXPERIMENTS else [])]
    tag = f".{os.getpid()}.tmp"

    def cc(src):
        obj = os.path.join(obj_dir, src.replace(".hip", ".o"))
        cmd = [HIPCC, *flags, *EXTRA_FLAGS.get(src, []), "-c", _src_path(src), "-o"]
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > _src_mtime(src) and _read(obj + ".cmd") == " ".join(cmd):
            return obj                                   # unchanged translation unit, same command: keep its object
        cmd.append(obj + tag)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr}")
        if r.stderr and (verbose or "-Wuninitialized" in r.stderr or "-Wreturn-type" in r.stderr or "-Wsometimes-uninitialized" in r.stderr):
            print(r.stderr, file=sys.stderr)         # these warnings have been real bugs: never hide them
        os.replace(obj + tag, obj)
        with open(obj + ".cmd" + tag, "w") as f:
            f.write(" ".join(cmd[:-1]))
        os.replace(obj + ".cmd" + tag, obj + ".cmd")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(cc, SOURCES))
    r = subprocess.run([HIPCC, *LINK_FLAGS, "-o", LIB_PATH + tag, *objs], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(LIB_PATH + tag, LIB_PATH)
    with open(STAMP_PATH + tag, "w") as f:
        f.write(_source_digest() + "\n")
    os.replace(STAMP_PATH + tag, STAMP_PATH)
    return LIB_PATH


def _read(path: str) -> str:
    try:
        with open(path) as f:
            return f.read()
    except OSError:
        return ""


def _src_mtime(src: str) -> float:
    """Newest mtime of a translation unit and every header it may include."""
    deps = [_src_path(src)] + [d for d in _all_deps() if d.endswith((".h", ".inc"))]
    return max(os.path.getmtime(d) for d in deps if os.path.exists(d))


class RzImageDesc(ctypes.Structure):
    """rz_image_desc (include/radzero_hip.h)"""
    _fields_ = [("image_dev", ctypes.c_void_p), ("src_dtype", ctypes.c_int32), ("height", ctypes.c_int32), ("width", ctypes.c_int32),
                ("channels", ctypes.c_int32), ("pad_left", ctypes.c_int32), ("pad_top", ctypes.c_int32), ("padded_height", ctypes.c_int32),
                ("padded_width", ctypes.c_int32), ("bounds_h_dev", ctypes.c_void_p), ("coeffs_h_dev", ctypes.c_void_p), ("ksize_h", ctypes.c_int32),
                ("bounds_v_dev", ctypes.c_void_p), ("coeffs_v_dev", ctypes.c_void_p), ("ksize_v", ctypes.c_int32)]


class RzConfig(ctypes.Structure):
    _fields_ = [
        ("compute_dtype", ctypes.c_int32), ("hidden_size", ctypes.c_int32), ("num_attention_heads", ctypes.c_int32),
        ("mlp_ratio", ctypes.c_int32), ("patch_size", ctypes.c_int32), ("num_channels", ctypes.c_int32),
        ("vit_layers", ctypes.c_int32), ("align_layers", ctypes.c_int32), ("vit_layer_norm_eps", ctypes.c_float),
        ("vocab_size", ctypes.c_int32), ("max_position_embeddings", ctypes.c_int32), ("text_layers", ctypes.c_int32),
        ("text_intermediate_size", ctypes.c_int32), ("text_layer_norm_eps", ctypes.c_float),
        ("pad_token_id", ctypes.c_int32), ("shared_layer_norm_eps", ctypes.c_float),
    ]


def _struct(name, doc, *fields):
    """A ctypes mirror of a C struct: "type name name ..." per line, types as in include/radzero_hip.h (i int32, f float, l int64, p pointer).
    `pack` makes the same bytes from the values in order (null pointers 0): a quarter of the time, for calls whose kernels are shorter than their host side."""
    t = {"i": ctypes.c_int32, "f": ctypes.c_float, "l": ctypes.c_int64, "p": ctypes.c_void_p}
    pack = struct.Struct("@" + "".join(f.split()[0].replace("l", "q").replace("p", "P") * (len(f.split()) - 1) for f in fields)).pack
    return type(name, (ctypes.Structure,), {"__doc__": doc, "_fields_": [(n, t[f.split()[0]]) for f in fields for n in f.split()[1:]], "pack": staticmethod(pack)})


RzRotaryArgs = _struct(
    "RzRotaryArgs", "rz_rotary_args (include/radzero_hip.h)",
    "i dtype layout batch tokens q_heads k_heads head_dim rotary_dim n_axes", "f amplitude",
    "p q_dev", "l q_batch_stride q_token_stride q_head_stride", "p k_dev", "l k_batch_stride k_token_stride k_head_stride",
    "p q_out_dev", "l q_out_batch_stride q_out_token_stride q_out_head_stride", "p k_out_dev", "l k_out_batch_stride k_out_token_stride k_out_head_stride",
    "p positions_dev", "l positions_batch_stride positions_token_stride", "p freqs_dev")
RzDiffAttentionArgs = _struct(
    "RzDiffAttentionArgs", "rz_diff_attention_args (include/radzero_hip.h)",
    "i dtype batch heads kv_heads n_q n_k head_dim causal", "f scale lambda_init norm_eps out_scale",
    "p q_dev", "l q_batch_stride q_token_stride q_head_stride", "p k_dev", "l k_batch_stride k_token_stride k_head_stride",
    "p v_dev", "l v_batch_stride v_token_stride v_head_stride", "p out_dev", "l out_batch_stride out_token_stride out_head_stride",
    "p lambda_qk_dev", "l lambda_head_stride", "p norm_weight_dev kv_lens_dev mask_dev", "l mask_batch_stride")
RzResidualNormArgs = _struct(
    "RzResidualNormArgs", "rz_residual_norm_args (include/radzero_hip.h)",
    "i dtype resid_dtype batch rows dim post_kind pre_kind", "f alpha post_eps pre_eps",
    "p y_dev", "l y_batch_stride y_row_stride", "p resid_dev", "l resid_batch_stride resid_row_stride",
    "p resid_out_dev", "l resid_out_batch_stride resid_out_row_stride", "p out_dev", "l out_batch_stride out_row_stride",
    "p post_weight_dev post_bias_dev scale_dev gate_dev", "l gate_batch_stride gate_row_stride", "p pre_weight_dev pre_bias_dev")


# every symbol include/radzero_hip.h declares: name -> (restype, argtypes)
_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
SYMBOLS = {
    "rz_last_error": (ctypes.c_char_p, []),
    "rz_version": (ctypes.c_char_p, []),
    "rz_create": (_I, [ctypes.POINTER(RzConfig), ctypes.POINTER(_P)]),
    "rz_destroy": (_I, [_P]),
    "rz_load_weight": (_I, [_P, ctypes.c_char_p, _P, _L]),
    "rz_weights_ready": (_I, [_P]),
    "rz_set_position_table": (_I, [_P, _I, _I, _P]),
    "rz_reserve": (_I, [_P, _I, _I, _I, _I]),
    "rz_padded_tokens": (_I, [_P, _I, _I, ctypes.POINTER(_I)]),
    "rz_vision_forward": (_I, [_P, _P, _I, _I, _I, _I, _P, _P]),
    "rz_text_forward": (_I, [_P, _P, _P, _I, _I, _P, _P, _P]),
    "rz_vlcabs": (_I, [_P, _P, _I, _I, _P, _P, _P, _P]),
    "rz_upsample_maps": (_I, [_P, _P, _L, _I, _I, _I, _I, _I, _P, _P]),
    "rz_grounding_points": (_I, [_P, _P, _L, _I, _I, _I, _I, _P, _P, _P]),
    "rz_grounding_points_ex": (_I, [_P, _P, _L, _I, _I, _I, _I, _I, _P, _P, _P]),
    "rz_upsample_maps_ex": (_I, [_P, _P, _L, _I, _I, _I, _I, _I, _I, _P, _P]),
    "rz_preprocess_image": (_I, [_P, _I, _I, _I, _I, _I, _P, _P, _I, _P, _P, _I, _P, _P, _F, _I, _P, _P, _P]),
    "rz_preprocess_batch_workspace": (ctypes.c_size_t, [ctypes.POINTER(RzImageDesc), _I, _I]),
    "rz_preprocess_batch": (_I, [ctypes.POINTER(RzImageDesc), _I, _I, _P, _P, _F, _I, _P, ctypes.c_size_t, _P, _P]),
    "rz_gemm": (_I, [_I, _I, _P, _P, _P, _P, _I, _I, _I, _P]),
    "rz_gemm_ex": (_I, [_I, _I, _P, _L, _P, _L, _P, _P, _L, _P, _P, _L, _I, _I, _I, _I, _I, _P]),
    "rz_gemm_qkv": (_I, [_I, _P, _P, _P, _P, _P, _I, _I, _I, _P, _P]),
    "rz_gemm_f32_split": (_I, [_I, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _P]),
    "rz_layernorm": (_I, [_I, _P, _P, _P, _F, _P, _P, _L, _I, _P]),
    "rz_flash_attention": (_I, [_I, _P, _P, _P, _P, _I, _I, _I, _I, _P]),
    "rz_flash_attention_split_workspace": (ctypes.c_size_t, [_I, _I, _I]),
    "rz_flash_attention_f32_split": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _I, _P]),
    "rz_flash_attention_f32_mx": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _I, _P]),
    "rz_text_embed_ln": (_I, [_I, _P, _P, _P, _P, _P, _F, _P, _P, _I, _I, _I, _I, _I, _P]),
    "rz_text_attention": (_I, [_I, _P, _P, _P, _P, _I, _I, _I, _P]),
    "rz_masked_meanpool": (_I, [_P, _P, _P, _I, _I, _I, _P]),
    "rz_rows_dot": (_I, [_P, _L, _P, _L, _P, _P, _I, _I, _I, _I, _L, _L, _L, _P]),
    "rz_image_features": (_I, [_P, _L, _I, _I, _I, _P, _P]),
    "rz_patch_embed": (_I, [_I, _P, _I, _I, _I, _I, _I, _P, _I, _P, _I, _P, _P, _P]),
    "rz_rotary": (_I, [ctypes.POINTER(RzRotaryArgs), _P]),
    "rz_diff_attention_workspace": (ctypes.c_size_t, [ctypes.POINTER(RzDiffAttentionArgs)]),
    "rz_diff_attention": (_I, [ctypes.POINTER(RzDiffAttentionArgs), _P, ctypes.c_size_t, _P]),
    "rz_residual_norm": (_I, [ctypes.POINTER(RzResidualNormArgs), _P]),
    "rz_set_option": (_I, [ctypes.c_char_p, _I]),
    "rz_set_model_option": (_I, [_P, ctypes.c_char_p, _I]),
    "rz_get_model_option": (_I, [_P, ctypes.c_char_p, ctypes.POINTER(_I)]),
    "rz_debug_buffer": (_I, [ctypes.c_char_p, _P]),
    "rz_profile_enable": (_I, [_P, _I]),
    "rz_profile_read": (_I, [_P, _P, _P]),
}

_lib = None


def load(auto_build: bool = True) -> ctypes.CDLL:
    """Load the shared library (building it first if the sources are newer and hipcc is present)."""
    global _lib
    if _lib is not None:
        return _lib
    # torch FIRST: its wheel bundles its own libamdhip64.so.7 / libhsa-runtime64.so.1 (same SONAMEs as /opt/rocm's).  Whichever copy is
    # mapped first serves the whole process; if this library pulled in /opt/rocm's before torch initialised the GPU through its own, the
    # process would hold two HIP runtimes and rz_create found no device (seen with `python __graft_entry__.py smoke`: build() then smoke()).
    import torch  # noqa: F401
    if auto_build and os.path.exists(HIPCC):
        build()
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"{LIB_PATH} is missing: run `python -c 'import __graft_entry__ as g; g.build()'`. "
            "radzero_amd has no CPU / PyTorch fallback.")
    lib = ctypes.CDLL(LIB_PATH)
    for name, (res, args) in SYMBOLS.items():
        fn = getattr(lib, name)           # AttributeError if the library does not export it
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


class RzError(RuntimeError):
    pass


def check(rc: int, what: str = ""):
    """Map C-ABI status codes to the exceptions the reference raises."""
    if rc == 0:
        return
    msg = load().rz_last_error().decode(errors="replace")
    if rc == 10001:
        raise ValueError(msg)
    if rc == 10003:
        raise NotImplementedError(msg)
    raise RzError(f"{what} failed with status {rc}: {msg}")
