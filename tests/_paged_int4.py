"""Inputs of the paged 4-bit cache's tests (CPU-side, seeded) and the tolerance of its attention."""
from __future__ import annotations

import numpy as np
import torch

from oracle import paged_int4_oracle as P

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def rounded(x: np.ndarray, dtype: str) -> np.ndarray:
    """x to the type and back (float64)."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(TYPES[dtype]).double().numpy()


def make_pool(pages, heads, dim, page_size, seed=0, outliers=True):
    """Random K and V (x8 channels in K), quantised: k_codes, k_params, v_codes, v_params."""
    rng = np.random.default_rng(seed)
    out = []
    for outlier in (outliers, False):
        x = rng.standard_normal((pages, heads, page_size, dim))
        if outlier:
            x[..., [c % dim for c in (7, 33)]] *= 8.0
        out += P.quantise(rounded(x, "fp16"))
    return out


def make_table(lens, page_size, seed=0, spare_pages=3, spare_columns=1):
    """Pages in no order: (table int32 [B, columns], pages in the pool); unused entries are -1."""
    needs = [-(-n // page_size) for n in lens]
    total = sum(needs) + spare_pages
    order = np.random.default_rng(seed + 1).permutation(total)
    table = np.full((len(lens), max(needs, default=0) + spare_columns), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(needs):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def tolerance(ref, mag, size, dim, dtype):
    """How far an output may be from the 64-bit one:

    * half a step of the output type;
    * the weights' rounding to fp16 for the second product, 2^-11 of each (and 2^-25 of the largest one for those
      below fp16's normal range: less than 2^-11 of a weight of 2^-14, and counted for 2^10 of them);
    * the scores: dim products summed in fp32 in any order, then scaled, reduced by the maximum and raised,
      4 more roundings (exp2 within 2 of its own): (dim + 8) 2^-24 of the sum of |q k| scale changes a weight by
      that share, and the sum of the weights too (factor 2); bf16 queries as fp16: 2^-25 of their largest element
      a channel, below dim 2^-24 of the sum that holds it with |k| of the same order (factor 2 once more);
    * the row sum and the products' accumulation in fp32: 2^-24 a term, below 2^-11 of the total for 2^12 terms."""
    half = torch.finfo(TYPES[dtype]).eps / 2
    scores = 2 * (2 if dtype == "bf16" else 1) * (dim + 8) * 2.0 ** -24 * size[..., None]
    return half * np.abs(ref) + (2.0 ** -11 + 2.0 ** -11 + scores) * mag + 2.0 ** -25
