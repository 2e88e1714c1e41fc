"""The logits head of include/et_logit_head.h in numpy float64, with the error its fp32 sums may have."""
from __future__ import annotations

import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of a rounding, relative to the value
SMALLEST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the smallest subnormal


def unpack(packed: np.ndarray, hidden: int) -> np.ndarray:
    n = np.empty((packed.shape[0], packed.shape[1] * 2), dtype=np.int64)
    n[:, 0::2], n[:, 1::2] = packed & 15, packed >> 4
    return n[:, :hidden]


def logits(x, packed, scales, zeros, group, out_dtype):
    """x [rows, hidden], packed [vocab, ceil(hidden / 2)], scales and zeros [vocab, groups] (float arrays).

    Returns (y, bound).  The bound counts roundings of 2^-24, each relative to the largest magnitude its sum
    can have at that place:
      * a group's products x (16 + n) are exact and are added to -24 sum x, itself added up in fp32: terms of at
        most 31 |x| and 24 |x|, in runs of at most min(group, 128) additions (accumulators start anew every 128
        columns) -- (min(group, 128) + 8) * 55 * |s| * sum |x| (8: the additions inside one product, in any order);
      * sum x, for the zeros, likewise: (min(group, 128) + 8) * |z| * sum |x|;
      * scaling and adding the runs up: one rounding per run and for each of the four parts of a row, relative to
        the sum of magnitudes;
      * the result's own rounding to its type, half a step."""
    x, scales = x.astype(np.float64), scales.astype(np.float64)
    zeros = np.zeros_like(scales) if zeros is None else zeros.astype(np.float64)
    hidden = x.shape[1]
    n = unpack(packed, hidden) - 8
    which = np.arange(hidden) // group
    w = n * scales[:, which] + zeros[:, which]
    y = x @ w.T
    run = min(group, 128)
    runs = -(-hidden // run) + 8
    ax = np.abs(x)
    inside = (run + 8) * (ax @ (55 * np.abs(scales) + np.abs(zeros))[:, which].T)
    outside = runs * (ax @ (np.abs(n * scales[:, which]) + np.abs(zeros[:, which])).T)
    bound = 2.0 ** -24 * (inside + outside)
    bound += HALF_STEP[out_dtype] * (np.abs(y) + bound) + SMALLEST[out_dtype]
    return y, bound
