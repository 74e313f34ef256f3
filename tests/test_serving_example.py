"""The serving example against a dense recomputation: every beam's last state from its whole history, in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def dense_state(model, history):
    """The last token's state of ``history`` with the whole sequence attended densely, in 64 bits."""
    h, kv, dim = model.heads, model.kv_heads, model.dim
    n = len(history)
    x = model.embedding[history].double()
    half = model.cos_sin.shape[1] // 2
    cos, sin = (model.cos_sin[:n, None, part].double() for part in (slice(0, half), slice(half, None)))

    def turn(y):
        a, b = y[..., :half], y[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
    for layer in range(model.layers):
        normal = x / (x.square().mean(-1, keepdim=True) + torch.finfo(model.dtype).eps).sqrt()
        qkv = (normal @ model.qkv[layer].double()).view(n, h + 2 * kv, dim)
        q, k, v = turn(qkv[:, :h]), turn(qkv[:, h:h + kv]), qkv[:, h + kv:]
        k, v = k.repeat_interleave(h // kv, 1), v.repeat_interleave(h // kv, 1)
        scores = torch.einsum("ihd,jhd->hij", q, k) * dim ** -0.5
        p = torch.softmax(scores.masked_fill(hidden, -torch.inf), -1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).flatten(1) @ model.out[layer].double()
    return x[-1]


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (3, 1, 128)])
def test_beams_match_a_dense_recomputation(heads, kv_heads, dim):
    from fgw_b200.examples.serving_step import Decoder, beam_decode
    model = Decoder(layers=2, heads=heads, kv_heads=kv_heads, dim=dim, vocab=97, positions=200)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(97, (n,), generator=gen).tolist() for n in (130, 1, 47)]
    tokens, scores, state = beam_decode(model, prompts, beams=3, steps=9)
    assert tokens.shape == (9, 9) and torch.isfinite(scores).all()
    for row in range(9):
        history = torch.tensor(prompts[row // 3] + tokens[row].tolist(), device="cuda")
        want = dense_state(model, history)
        # about a dozen BF16 roundings (2^-8 each at most, independent) between the embedding and the state
        off = (state[row].double() - want).norm() / want.norm()
        assert off <= 12 * 2.0 ** -8, (row, off.item())
    # the beams of a prompt are different continuations
    for p in range(3):
        assert len({tuple(t) for t in tokens[3 * p:3 * p + 3].tolist()}) == 3
