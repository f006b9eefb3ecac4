"""Row copies and the operations behind them: attention over 16-bit pages and short convolutions read what earlier steps left ahead of
their wait for the kernel in front, and the rows of a copy are to lie there by then."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_copies_attention_and_convolution_one_right_behind_the_other():
    """Eight requests forked and stepped on, over other rows every time, without a pause: equal to the same with one."""
    from types import SimpleNamespace

    from gibbs_b200 import ops
    n, heads, kv_heads, hd, page, blocks, hidden, taps = 8, 32, 8, 64, 16, 65, 2048, 3
    gen = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(DEV)                        # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                                     # noqa: E731
    sources = [(rand(n * blocks, kv_heads, page, hd), rand(n * blocks, kv_heads, page, hd), rand(n, taps - 1, hidden).float()) for _ in range(6)]
    k, v = (torch.zeros(2 * n * blocks, kv_heads, page, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    state = torch.zeros(2 * n, taps - 1, hidden, device=DEV)
    copies = ops.RowCopies([[k, v], [state]])
    pairs = [[(i, n * blocks + i) for i in range(n * blocks)], [(i, n + i) for i in range(n)]]
    bt = (torch.arange(n * blocks, dtype=torch.int32).view(n, blocks) + n * blocks).to(DEV)
    length = blocks * page - 1                                     # positions that earlier steps filled
    hints = SimpleNamespace(n_tokens=n, n_requests=n, q_start=i32(list(range(n))), q_len=i32([1] * n), start_pos=i32([length] * n),
                            max_q_len=1, max_ctx_len=length + 1, status=ops.device_status(torch.device(DEV)))
    qkv, bcx = rand(n, (heads + 2 * kv_heads) * hd), rand(n, 3 * hidden)
    weight = torch.randn(hidden, taps, generator=gen).to(DEV)
    slots, tok_req, tok_pos = i32(list(range(n, 2 * n))), i32(list(range(n))), i32([length] * n)
    out = torch.empty(n, heads * hd, dtype=torch.bfloat16, device=DEV)
    conv = torch.empty(n, hidden, dtype=torch.bfloat16, device=DEV)

    def run(pause):
        got = []
        for sk, sv, ss in sources:
            k[:n * blocks], v[:n * blocks], state[:n] = sk, sv, ss
            pause()
            copies.copy(pairs)
            pause()
            ops.qk_norm_rope_store(qkv, heads, kv_heads, hd, None, None, 1e-5, None, 0, False, tok_req, tok_pos, bt, k, v, hints.status)
            pause()
            ops.paged_attention(qkv[:, :heads * hd], heads, kv_heads, hd, k, v, bt, tok_req, tok_pos, hd ** -0.5, 0, out, hints.status, hints=hints)
            got.append(out.clone())
            pause()
            state[:n] += 1
            pause()
            copies.copy([[], pairs[1]])
            pause()
            ops.short_conv(bcx, weight, None, state, slots, tok_req, hints.q_start, hints.q_len, conv, 1)
            got.append(conv.clone())
            got.append(state.clone())
        torch.cuda.synchronize()
        return got

    want = run(torch.cuda.synchronize)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), want))
    assert int(hints.status.item()) == 0


@pytest.mark.parametrize("pairs", [[(0, 1, 2), (3,)], [(0, 1), (2,)], [(0, 1, 2, 3)], [(), (0, 1, 2, 3)], [0, 1], [("0", "1")], [(0.0, 1.0)], [(None, 1)],
                                   [[[0, 1], [2, 3]]]])
def test_pairs_that_are_not_pairs_are_refused(pairs):
    from gibbs_b200.ops import KernelError, RowCopies
    t = torch.arange(40, device=DEV).float().view(10, 4)
    before, copies = t.clone(), RowCopies([[t], [t.clone()]])
    for given in ([pairs, []], [[], pairs]):
        with pytest.raises(KernelError, match="row copies"):
            copies.copy(given)
    assert torch.equal(t, before)
    assert copies.copy([[], [[1, 0]]]) == 1 and copies.copy([[(3, 2)], []]) == 1
    assert torch.equal(t[2], t[3])
