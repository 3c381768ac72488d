"""The 64-bit forms against tiny cases worked out by their definition."""
import math

import torch

from sequence_oracle import attend64, linear64, rotate64, seen


def test_seen_by_hand():
    # 2 queries, the last of 5 keys; one to the left, none to the right, one sink
    assert seen(2, 5, 1, 0, 1).tolist() == [[True, False, True, True, False],
                                            [True, False, False, True, True]]
    # more queries than keys: the first stand before every key
    assert seen(3, 1, None, 0, 4).tolist() == [[False], [False], [True]]
    assert seen(2, 2, None, None, 0).all()


def test_attention_by_hand():
    q = torch.tensor([[[1.0]], [[2.0]]])
    k = torch.tensor([[[0.5]], [[-1.0]], [[math.nan]]])
    v = torch.tensor([[[3.0]], [[5.0]], [[math.inf]]])
    # causal; the third key belongs to a second sample, which has no queries
    out, _ = attend64(q, k, v, [2, 0], [2, 1], (None, 0), 0, scale=1.0)
    a, b = math.exp(1.0), math.exp(-2.0)
    assert abs(out[0, 0, 0].item() - 3.0) < 1e-12
    assert abs(out[1, 0, 0].item() - (a * 3 + b * 5) / (a + b)) < 1e-12


def test_rotation_by_hand():
    x = torch.tensor([[[3.0, 4.0, 0.0, 0.0]]])
    out, _ = rotate64(x, torch.tensor([[2]], dtype=torch.int32), eps=0.0, base=100.0)
    # two pairs on one axis: (3, 0) by 2 rad, (4, 0) by 2 / 10 rad; norm sqrt(25 / 4)
    want = [3 * math.cos(2), 4 * math.cos(0.2), 3 * math.sin(2), 4 * math.sin(0.2)]
    assert torch.allclose(out[0, 0], torch.tensor(want, dtype=torch.float64) / 2.5, atol=1e-12)


def test_linear_by_hand():
    out, _ = linear64(torch.tensor([[1.0, 2.0]]), torch.tensor([[3.0, -1.0], [-1.0, 0.0]]),
                      torch.tensor([1.0, -1.0]), "relu", torch.tensor([[10.0, 20.0]]))
    assert out.tolist() == [[12.0, 20.0]]
    for act, want in (("gelu", 0.5 * (1 + math.erf(1 / math.sqrt(2)))),
                      ("silu", 1 / (1 + math.exp(-1))),
                      ("gelu_tanh", 0.5 * (1 + math.tanh(math.sqrt(2 / math.pi) * 1.044715)))):
        got, _ = linear64(torch.ones(1, 1), torch.ones(1, 1), act=act)
        assert abs(got.item() - want) < 1e-12, act
