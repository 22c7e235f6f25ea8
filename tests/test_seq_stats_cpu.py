"""The work of packed sequences, by counting: what Stats says of the paged cache and packed attention."""
import random

import pytest
import torch


@pytest.fixture(autouse=True)
def no_graph(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


@pytest.mark.parametrize("seed", range(20))
def test_flops(srdit, seed):
    rng = random.Random(seed)
    B, T = rng.randint(0, 5), rng.randint(0, 40)
    cu = [rng.randint(-3, T + 3) for _ in range(B + 1)]
    if seed % 2:
        cu.sort()
    lens = [rng.randint(0, 30) for _ in range(B)]
    for causal in (True, False):
        work = srdit.ops._attn_flops((T, 3, 8), B, torch.tensor(cu, dtype=torch.int32), lambda: lens,
                                     causal)
        seen = 0
        for b, L in enumerate(lens):
            lo, hi = (min(max(x, 0), T) for x in cu[b:b + 2])
            n = max(hi - lo, 0)
            seen += sum(min(max(L - n + i + 1, 0), L) if causal else L for i in range(n))
        assert work() == 4 * 3 * 8 * seen


def test_flops_and_bytes_of_equal_sequences(srdit):
    assert srdit.ops._attn_flops((6, 1, 8), 2, None, lambda: [3, 5], False)() == 4 * 8 * 3 * 8
    bf16 = torch.bfloat16
    assert srdit.ops._kv_bytes(7, 3, None, 2, 16, bf16, torch.int8)() == 6 * 2 * 2 * (32 + 16 + 4)
    cu = torch.tensor([1, 3, 4], dtype=torch.int32)
    assert srdit.ops._kv_bytes(7, 2, cu, 2, 16, bf16, bf16)() == 3 * 2 * 2 * (32 + 32)
