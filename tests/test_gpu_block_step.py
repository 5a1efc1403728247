"""``MurmurativeBlock.step`` is the block's own function: all of its rounds, for any number of them."""
import pytest
import torch

from murmurative_attention_b200 import MurmurativeBlock
from test_gpu_block import TOL

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rounds", [None, 0, 1, 2, 5])
def test_first_step_is_forward_on_one_token(rounds, causal):
    """A fresh pool and one token: the same selections, updates and sums (fp32, so that the pool's rounding
    is forward's). None: the default rounds."""
    torch.manual_seed(3)
    B, D, H = 3, 64, 4
    kw = dict() if rounds is None else dict(rounds=rounds)
    block = MurmurativeBlock(D, H, slots=32, causal=causal, device="cuda", dtype=torch.float32, **kw)
    x = torch.randn(B, D, device="cuda")
    pool = block.new_pool(B)
    before = pool.keys.clone()
    y = block.step(x, pool)
    with torch.no_grad():
        want = block(x.unsqueeze(1), torch.zeros(B, 1, dtype=torch.int64, device="cuda"))[:, 0]
    torch.testing.assert_close(y, want, **TOL)
    assert torch.equal(pool.positions.cpu(), torch.ones(B, dtype=torch.int64))  # one token, whatever the rounds
    assert torch.equal(pool.keys, before) == (rounds == 0)


def test_rounds_of_a_step_are_steps_of_the_pool():
    """Several tokens, against the pool driven by hand."""
    torch.manual_seed(4)
    B, D, H = 2, 64, 4
    block = MurmurativeBlock(D, H, slots=32, rounds=3, causal=True, device="cuda", dtype=torch.float32)
    pool, hand = block.new_pool(B), block.new_pool(B)
    for t in range(5):
        x = torch.randn(B, D, device="cuda")
        y = block.step(x, pool)
        q = block._queries(block.norm1(x).unsqueeze(1), hand.positions.unsqueeze(1))[:, :, 0].detach()
        attn = 0
        for _ in range(3):
            attn = attn + hand.step(q, q, q, causal=True, gamma=0.15)
            hand.positions -= 1
        hand.positions += 1
        h = x + attn.reshape(B, D) @ block.o_proj.weight.t()
        f = torch.nn.functional.gelu(block.norm2(h) @ block.up.weight.t() + block.up.bias)
        torch.testing.assert_close(y, h + f @ block.down.weight.t() + block.down.bias, **TOL)
        assert torch.equal(pool.keys, hand.keys) and torch.equal(pool.positions, hand.positions)
