"""ctypes binding of libtvae_hip.so (C ABI: include/tvae_hip.h).

The library is built in-tree by ``build()`` (``make`` in csrc/, hipcc --offload-arch=gfx950)
and loaded lazily.  There is NO fallback: if the shared object is missing or a call fails
the caller gets a RuntimeError — the product path never routes through a CPU
implementation.
"""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
LIB_PATH = os.path.join(_HERE, "libtvae_hip.so")
HOST_PATH = os.path.join(_HERE, "_host.so")         # C++ autograd nodes over the library (csrc/host.cpp)
HEADER = os.path.join(os.path.dirname(_HERE), "include", "tvae_hip.h")

TVAE_F32, TVAE_BF16, TVAE_F32_STRICT = 0, 1, 2      # TVAE_F32_STRICT: tvae_mmd_* only (include/tvae_hip.h)
TVAE_F16 = 3                                        # tvae_dropout and tvae_norm_* only
TVAE_NORM_LAYER, TVAE_NORM_RMS = 0, 1

_i64, _vp, _int, _f32, _f64 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_double
_u64 = ctypes.c_uint64

# name -> (restype, argtypes); mirrors include/tvae_hip.h one to one
SIGNATURES = {
    "tvae_version": (_int, []),
    "tvae_last_error": (ctypes.c_char_p, []),
    "tvae_encode_fwd_workspace_bytes": (_i64, [_i64] * 4),
    "tvae_encode_fwd": (_int, [_vp, _i64, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64, _vp]),
    "tvae_encode_bwd_workspace_bytes": (_i64, [_i64] * 4),
    "tvae_encode_bwd": (_int, [_vp, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _int,
                               _vp, _i64, _vp]),
    "tvae_encode_bwd_sum": (_int, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64,
                                   _int, _vp, _i64, _vp]),
    "tvae_decode_fwd_workspace_bytes": (_i64, [_i64] * 3),
    "tvae_decode_fwd": (_int, [_vp, _vp, _vp, _vp, _vp, _f32, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _int, _vp, _i64,
                               _vp]),
    "tvae_decode_bwd_workspace_bytes": (_i64, [_i64] * 3),
    "tvae_decode_bwd": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _int,
                               _vp, _i64, _vp]),
    "tvae_mmd_workspace_bytes": (_i64, [_i64, _i64, _i64, _int]),
    "tvae_mmd_workspace_bytes_for": (_i64, [_i64, _i64, _i64, _int, _int]),
    "tvae_profile_next_mmd": (_int, [_vp, _vp]),
    "tvae_upsample_out_len": (_i64, [_i64, _i64, _i64, _int, _int]),
    "tvae_upsample_fwd": (_int, [_vp, _vp, _i64, _i64, _i64, _i64, _i64, _int, _int, _int, _vp]),
    "tvae_upsample_bwd": (_int, [_vp, _vp, _i64, _i64, _i64, _i64, _i64, _int, _int, _int, _vp]),
    "tvae_slerp": (_int, [_vp, _vp, _vp, _f32, _vp, _i64, _i64, _int, _vp]),
    "tvae_rbf_kernel_fwd": (_int, [_vp, _vp, _i64, _i64, _i64, _vp, _vp]),
    "tvae_rbf_kernel_bwd": (_int, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _vp, _vp, _vp]),
    "tvae_mmd_fwd_bwd": (_int, [_vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _vp, _f64, _vp, _f64, _vp, _i64, _vp]),
    "tvae_mmd_shard_layout": (_int, [_i64, _i64, _i64, _int, _int, _vp]),
    "tvae_mmd_stats_local": (_int, [_vp, _vp, _i64, _i64, _i64, _i64, _int, _int, _vp, _i64, _vp]),
    "tvae_mmd_prep_local": (_int, [_vp, _vp, _i64, _i64, _i64, _i64, _int, _int, _vp, _i64, _vp]),
    "tvae_mmd_tiles": (_int, [_vp, _i64, _i64, _i64, _i64, _int, _vp, _vp, _f64, _vp, _f64, _int, _vp, _i64, _vp]),
    "tvae_mmd_fwd_bwd_static": (_int, [_vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _vp, _f64, _vp, _f64, _vp]),
    "tvae_small_step_supported": (_int, [_i64] * 4),
    "tvae_small_step_fwd_workspace_bytes": (_i64, [_i64] * 4),
    "tvae_small_step_bwd_workspace_bytes": (_i64, [_i64] * 4),
    # h, stride_b, stride_s, We, be, Wd, bd, gamma, beta, eps, prior, B, n_eff, d, L, dtype, latent, recon, pre, mean, rstd,
    # d_latent_mmd, sums3, loss, loss_scale, grad_scale, workspace, bytes, stream
    "tvae_small_step_fwd": (_int, [_vp, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _f32, _vp, _i64, _i64, _i64, _i64, _int,
                                   _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _f64, _f64, _vp, _i64, _vp]),
    # d_recon, d_reg, latent, pre, mean, rstd, gamma, Wd, We, h, stride_b, stride_s, d_latent_mmd, dh, dWe, dbe, dWd, dbd,
    # dgamma, dbeta, B, S, n_eff, d, L, dtype, workspace, bytes, stream
    "tvae_small_step_bwd": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _vp,
                                   _vp, _vp, _i64, _i64, _i64, _i64, _i64, _int, _vp, _i64, _vp]),
    # in, so, si, residual, so, si, grp, out, rows, d, p, rng, seed, offset, in_dtype, out_dtype, stream
    "tvae_dropout": (_int, [_vp, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _i64, _f64, _vp, _u64, _u64, _int, _int, _vp]),
    # kind, x, so, si, residual, so, si, grp, weight, bias, eps, p, rng, seed, offset, y, sum, mean, rstd, rows, d, dtype,
    # w_dtype, r_dtype, stream
    "tvae_norm_fwd": (_int, [_int, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _f64, _f64, _vp, _u64, _u64, _vp, _vp, _vp,
                             _vp, _i64, _i64, _int, _int, _int, _vp]),
    "tvae_norm_bwd_workspace_bytes": (_i64, [_i64] * 2),
    # kind, dy, so, si, dsum, so, si, x, so, si, residual, so, si, grp, weight, mean, rstd, p, rng, seed, offset, dx, dresidual,
    # dweight, dbias, rows, d, dtype, w_dtype, r_dtype, workspace, bytes, stream
    "tvae_norm_bwd": (_int, [_int, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _f64,
                             _vp, _u64, _u64, _vp, _vp, _vp, _vp, _i64, _i64, _int, _int, _int, _vp, _i64, _vp]),
}

_lock = threading.Lock()
_lib = None
_host = None


def build(force: bool = False) -> str:
    """Compile csrc/*.hip into libtvae_hip.so for gfx950 and csrc/host.cpp into _host.so.  Works without a GPU."""
    if force:
        subprocess.run(["make", "-C", CSRC, "clean"], check=True, capture_output=True)
    proc = subprocess.run(["make", "-C", CSRC, "-j4", "all", "host", f"PYTHON={sys.executable}"], capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("building libtvae_hip.so failed:\n" + proc.stdout + proc.stderr)
    return LIB_PATH


def lib() -> ctypes.CDLL:
    """The loaded library (loads on first use; raises if it has not been built)."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                if not os.path.exists(LIB_PATH):
                    raise RuntimeError(
                        f"{LIB_PATH} is missing: the HIP extension has not been built "
                        "(run `python -c 'import __graft_entry__ as g; g.build()'` or `make -C transformer_vae_amd/csrc`). "
                        "There is no CPU fallback for this path.")
                handle = ctypes.CDLL(LIB_PATH)
                for name, (res, args) in SIGNATURES.items():
                    fn = getattr(handle, name)
                    fn.restype = res
                    fn.argtypes = args
                _lib = handle
    return _lib


def host():
    """The module of C++ autograd nodes (loads on first use; raises if it has not been built)."""
    global _host
    if _host is None:
        if not os.path.exists(HOST_PATH):
            raise RuntimeError(f"{HOST_PATH} is missing: the extension has not been built "
                               "(run `python -c 'import __graft_entry__ as g; g.build()'` or `make -C transformer_vae_amd/csrc all host`). "
                               "There is no CPU fallback for this path.")
        handle = lib()._handle          # before the module: the other way round a call costs 0.6 us more host time (4.4 and 5.0)
        from . import _host as module
        module.bind(handle)
        _host = module
    return _host


def check(status: int, what: str) -> None:
    if status != 0:
        msg = lib().tvae_last_error()
        raise RuntimeError(f"{what} failed (status {status}): {msg.decode() if msg else 'unknown error'}")
