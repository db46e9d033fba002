"""Exponents of the 8-bit cache's attention for logits of any size: a float32 model of a step (no GPU).

A step takes P = 2^y against a maximum m of earlier steps, y a fused multiply-add, and where P grows past what
float16 sums hold it takes m anew and P from the differences of the rounded logits.
"""

from __future__ import annotations

import os
import re

import numpy as np
import pytest

import mini_vllm_b200

CSRC = os.path.join(os.path.dirname(mini_vllm_b200._native.__file__), "csrc")
F32, LIMIT = np.float32, 16384.0


def fused(s, f, m, ve):
    """fma(s, f, ve - m): the product is exact in 64 bits."""
    return (s.astype(np.float64) * np.float64(f) + np.float64(F32(ve - m))).astype(F32)


def differences(s, f, m, ve):
    return ((s * f).astype(F32) - (F32(0) if m == -np.inf else m)).astype(F32) + F32(ve)


def step(s, f, m, ve):
    """(P, the new maximum, passes over the scores)."""
    if m > -np.inf:
        with np.errstate(over="ignore"):
            p = np.exp2(fused(s, f, m, ve).astype(np.float64))
        if not (p > LIMIT / 2).any():  # (a sum of two of them: the smallest that the kernels look at)
            return p, m, 1
    m = max(m, (s * f).astype(F32).max())
    return np.exp2(differences(s, f, m, ve).astype(np.float64)), m, 2


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("ve", [-4.0, 0.0, 0.7, 7.0])
def test_a_step_ends_with_its_largest_key_kept(sign, ve):
    r = np.random.RandomState(int(10 * ve) + sign + 50)
    beyond = 0
    for e in range(0, 41):
        for _ in range(40):
            s = (sign * r.uniform(1.0, 4.0, 64) * 2.0 ** 10).astype(F32)
            f = F32(r.uniform(1.0, 2.0) * 2.0 ** (e - 11))
            p, m, passes = step(s, f, F32(-np.inf), ve)
            assert passes == 2 and m == (s * f).astype(F32).max()
            y = differences(s, f, m, ve)
            assert y.max() == F32(ve) and p.max() == 2.0 ** float(F32(ve)) and 16 * p.max() < LIMIT
            again, m2, _ = step(s, f, m, ve)  # the same scores once more, against their own maximum
            assert m2 == m and (again <= LIMIT).all()
            beyond += (np.exp2(np.minimum(fused(s, f, m, ve), 100).astype(np.float64)) > LIMIT).any()
            more, m3, _ = step((s * F32(1 + sign * 0.5)).astype(F32), f, m, ve)
            assert m3 >= m and (more <= LIMIT).all()
            if m3 > m + 16:
                assert more.max() == 2.0 ** float(F32(ve))
    assert beyond > 0  # the fused form alone passes the limit against the very maximum


def test_products_that_overflow():
    s, f = np.full(16, -3e38, F32), F32(4.0)
    with np.errstate(over="ignore"):
        p, m, passes = step(s, f, F32(-np.inf), 0.0)
        assert m == -np.inf and passes == 2 and (p == 0).all()
        s[3] = 1.0
        p, m, _ = step(s, f, m, 0.0)
    assert m == 4.0 and p[3] == 1.0 and p.sum() == 1.0


@pytest.mark.parametrize("source", ["fp8_decode.cu", "fp8_prefill.cu"])
def test_every_loop_has_a_bound_in_its_head(source):
    text = open(os.path.join(CSRC, source)).read()
    assert not re.search(r"for \([^;]*;\s*;|while \((true|1)\)", text)


def test_the_inputs_have_winners_and_the_logits_they_say():
    import torch

    import fp8_large_logits as L
    import fp8_model as F

    for name, (_, _, _, _, sign) in L.CASES.items():
        for heads in L.HEADS:
            spans = [(n, 1) for n in (700, 1, 40, 17, 333)]
            q, kc, vc, sc, table, scale = L.case(name, spans, heads, 16)
            assert torch.isfinite(q.float()).all()
            for i, (n, _) in enumerate(spans):
                _, sure, _ = L.winners(q[i:i + 1], kc, vc, sc, table[i], n, 16, scale)
                assert sure.all()
                k = F.dequant(kc, sc, 0, table[i, :-(-n // 16)], n).repeat_interleave(heads[0] // heads[1], 0)
                x = torch.matmul(q[i].double()[:, None], k.transpose(1, 2)) * scale * 1.4426950408889634
                top = x.amax(-1)
                assert (top.abs() >= 2.0 ** 23).all() and (top.abs() <= 2.0 ** 43).all()
                assert (torch.sign(top) == (1 if sign * scale > 0 else -1)).all()


def test_most_rows_of_chunks_have_winners():
    import fp8_large_logits as L

    for name in L.CASES:
        for spans in ([(700, 700), (1, 1), (300, 200)], [(2100, 20), (50, 3), (17, 1)]):
            for heads in L.HEADS[:2]:
                q, kc, vc, sc, table, scale = L.case(name, spans, heads, 16)
                at = 0
                for i, (n, rows) in enumerate(spans):
                    _, sure, _ = L.winners(q[at:at + rows], kc, vc, sc, table[i], n, 16, scale)
                    assert sure.double().mean() > 0.9
                    at += rows
