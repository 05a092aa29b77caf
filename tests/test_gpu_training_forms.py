"""Sizes that reach every kernel of the training operators; tests/test_training_forms.py
asks the rules, on the host, that they do."""
from __future__ import annotations

import pytest

import test_gpu_cross_entropy as entropy
import test_gpu_gated_recurrence as recurrence
from training_reference import TYPES, cross_entropy, cross_entropy_backward

pytestmark = pytest.mark.gpu

# m x n x k of products, by tile: several steps of k and a part of one.
TILES = {
    "bf16": {"k256x256": [(2600, 3100, 200)], "k128x128": [(1030, 2050, 1100)], "k64x128": [(1030, 2050, 200)],
             "k64x64": [(500, 2050, 200), (4100, 200, 200)], "k32x64": [(20, 40, 520), (3100, 130, 200)]},
    "f32": {"k256x256": [(3100, 4100, 200)], "k128x128": [(1500, 2050, 200)], "k64x128": [(2050, 2600, 200)],
            "k64x64": [(500, 2050, 200), (4100, 200, 200)], "k32x64": [(20, 40, 520)]},
}
# The same where k is cut into parts.
PARTS = {"bf16": {"k128x128": [(1500, 130, 9000)], "k64x128": [(40, 2050, 4200)], "k64x64": [(2050, 40, 4200)],
                  "k32x64": [(20, 20, 2100), (40, 2050, 2100)]},
         "f32": {"k128x128": [(3100, 200, 4200)], "k64x64": [(130, 200, 9000)],
                 "k32x64": [(20, 20, 1100), (2050, 20, 2100)]}}
# What m, n and k are: rows, vocabulary and width of the logits, of the two gradients.
ROLES = {"logits": lambda m, n, k: (m, n, k), "grad_x": lambda m, n, k: (m, k, n), "grad_weight": lambda m, n, k: (k, m, n)}
RECURRENCES = {
    "kOne": [(3, 1, 130), (2, 1, 65)], "kFew": [(2, 20, 130), (2, 30, 65)],
    "kMany": [(2, 60, 64), (2, 50, 33), (170, 200, 64)], "kLong": [(170, 200, 64), (170, 200, 33)],
    "parts": [(1, 1000, 130), (2, 700, 33)]}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("role", ROLES)
@pytest.mark.parametrize("tile", list(TILES["f32"]))
def test_products(device, dtype, role, tile):
    sizes = TILES[dtype][tile] + PARTS[dtype].get(tile, [])
    for size in sizes:
        x, w, targets, grad = entropy.operands(TYPES[dtype], *ROLES[role](*size), seed=sum(size))
        got = entropy.forward(device, x, w, targets)
        entropy.check(got, cross_entropy(x, w, targets))
        entropy.check(entropy.backward(device, x, w, targets, got["lse"], grad),
                      cross_entropy_backward(x, w, targets, got["lse"], grad))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", RECURRENCES)
def test_recurrences(device, dtype, form):
    for size in RECURRENCES[form]:
        recurrence.check_both(device, *recurrence.operands(TYPES[dtype], *size, seed=sum(size)))
