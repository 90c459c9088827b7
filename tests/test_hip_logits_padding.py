"""Logits' rules over padded trees: nodes at or past a sequence's count are on
no path, whatever their bits and drafted tokens say (attention over the INT8
cache, which takes the same tree and counts, ignores them too)."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_attention_q8 import words_of
from test_hip_logits_rules import ALL, expect, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,counts", [(6, [6, 0, -3, 2, 99]), (5, [1, 4, 5, 2, 3]), (70, [65, 64, 1, 66, 70])])
@pytest.mark.parametrize("use", [ALL, ("drafted", "tree", "presence", "frequency")], ids="+".join)
def test_bits_of_padding_nodes_are_ignored(hip, rows, counts, use):
    a = inputs(len(counts), rows, 2500, 100, 8, 0, rows)
    a["tree"] = words_of(np.ones((len(counts), rows, rows), bool))   # every node on every path
    a["tree"] |= np.uint64(0xffffffffffffffff)                        # and what lies past the rows
    print(f"case logits padding nodes rows={rows} {counts}", flush=True)
    got, tokens = run(hip, a, use, 0, counts=counts)
    for s, c in enumerate(counts):
        c = max(0, min(rows, c))
        a["sees"] = np.zeros((len(counts), rows, rows), bool)
        a["sees"][:, :, :c] = True
        want, wt = expect(a, use, 0)
        assert np.array_equal(got[s, :c], want[s, :c]) and np.array_equal(tokens[s, :c], wt[s, :c]), s
        assert (got[s, c:] == 7.0).all() and (tokens[s, c:] == 77).all()
