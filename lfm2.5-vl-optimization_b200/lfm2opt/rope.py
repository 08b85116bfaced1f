"""Frequency tables of rotary positions, for the kernels that turn heads by positions * inv_freq (qk_norm_rope_kv,
qk_norm_rope_kv_paged). Computed once at load time, in fp64, and rounded to fp32.

    inv_freq(rot_dim, theta)                                     theta^(-2 i / rot_dim), i < rot_dim / 2
    inv_freq(..., kind="linear", factor=4)                       positions stretched: every frequency / factor
    inv_freq(..., kind="ntk", factor=4)                          theta grown so that the slowest pair turns 1 / factor as
                                                                 fast and the fastest as before
    inv_freq(..., kind="yarn", factor=4, original=8192)          fast pairs (more than beta_fast turns over the original
                                                                 length) kept, slow ones (fewer than beta_slow) divided
                                                                 by factor, a linear ramp over the pairs between; scaling
                                                                 0.1 ln(factor) + 1
    inv_freq(..., kind="llama3", factor=8, original=8192)        wavelengths below original / high_freq kept, above
                                                                 original / low_freq divided by factor, between them
                                                                 interpolated in original / wavelength
"""

import math

import torch


def inv_freq(rot_dim, theta=1e6, kind="plain", factor=1.0, original=None, beta_fast=32.0, beta_slow=1.0,
             low_freq=1.0, high_freq=4.0, device=None):
    """(inv_freq fp32 [rot_dim / 2], scaling): the table and the factor on the cosines and sines that the kernels take."""
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError("rot_dim must be positive and even")
    if factor < 1.0:
        raise ValueError("factor must be >= 1")
    if kind in ("yarn", "llama3") and (original is None or original <= 0):
        raise ValueError(f"{kind} needs original, the length the model was trained on")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim
    scaling = 1.0
    if kind == "ntk":
        if rot_dim <= 2:
            raise ValueError("ntk needs rot_dim > 2")
        theta = theta * factor ** (rot_dim / (rot_dim - 2))
    f = theta ** -i
    if kind == "linear":
        f = f / factor
    elif kind == "yarn":
        def pair(turns):  # the (real) pair index that makes `turns` turns over the original length
            return rot_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rot_dim - 1)
        ramp = ((torch.arange(rot_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        scaling = 0.1 * math.log(factor) + 1.0
    elif kind == "llama3":
        turns = original * f / (2 * math.pi)  # original / wavelength
        mid = ((turns - low_freq) / (high_freq - low_freq)).clamp(0, 1)
        f = f / factor * (1 - mid) + f * mid
    elif kind not in ("plain", "ntk"):
        raise ValueError(f"unknown kind {kind!r}: plain, linear, ntk, yarn or llama3")
    return f.float().to(device) if device is not None else f.float(), scaling
