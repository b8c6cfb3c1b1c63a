"""The text decoder example (ppocr_b200.textgen) against a plain fp32 decoder
that quantises its keys and values as the cache does."""

import math

import pytest
import torch

from oracle import decode as O

pytestmark = pytest.mark.gpu

F16 = torch.float16


class Plain:
    """The same decoder on the CPU in fp32, rounded to fp16 where the decoder
    stores a tensor. It attends to what the decoder's caches hold (a key or
    value whose last bit differs would fall on another code now and then, a
    whole quantisation step apart), after checking it against its own keys and
    values."""

    def __init__(self, dec, w, sequence):
        self.s, self.dec, self.b = dec.shape, dec, sequence
        f = lambda t: t.float().cpu()  # noqa: E731
        self.w = {k: [f(t) for t in v] if isinstance(v, list) else f(v) for k, v in vars(w).items()}

    def run(self, x):
        """x [n, dim]: the sequence's last n embeddings, which the decoder has
        taken in; logits [n, vocab]."""
        s, w, dec = self.s, self.w, self.dec
        held = lambda x: x.half().float()  # noqa: E731
        norm = lambda x: held(torch.nn.functional.layer_norm(x, (s.dim,), eps=1e-5))  # noqa: E731
        length = int(dec.lengths[self.b])
        x = held(x)
        for n in range(s.layers):
            qkv = held(norm(x) @ w["qkv"][n].T)
            q, k, v = qkv.split([s.heads * s.head_dim] + [s.kv_heads * s.head_dim] * 2, 1)
            cache, cached = dec.caches[n], []
            for which, y in ((0, k), (1, v)):
                got = O.held(cache.pool.cpu(), cache.page_size, s.head_dim, F16, dec.table[self.b].cpu(), length, which)
                y = y.unflatten(1, (s.kv_heads, -1))
                _, step, _ = O.quantise(y.half())
                off = (got[length - x.shape[0]:] - y).abs().unflatten(-1, (-1, 32)).amax(-1)
                assert (off <= 1.5 * step.double() + 0.05).all()
                cached.append(got)
            o, _, _ = O.attention(q.unflatten(1, (s.heads, -1)), *cached, length - x.shape[0], s.head_dim ** -0.5,
                                  s.window, s.sinks)
            x = held(held(held(o.float()).flatten(1) @ w["out"][n].T) + x)
            up = held(torch.nn.functional.silu(held(norm(x) @ w["up"][n].T)))
            x = held(held(up @ w["down"][n].T) + x)
        return (norm(x) @ w["head"].T)[:, : s.vocab]


@pytest.mark.parametrize("window,sinks", [(0, 0), (12, 2)])
def test_decoder_logits(native, cuda, window, sinks):
    """Prompts of different lengths, then single tokens; relative L2 2e-2, the
    framework's largest bar for fp16 storage (its max-abs bar)."""
    from ppocr_b200 import textgen

    shape = textgen.DecoderShape(inputs=120, vocab=1003, dim=256, heads=4, kv_heads=2, mlp=512, window=window,
                                 sinks=sinks)
    w = textgen.DecoderWeights(shape, cuda, positions=64, seed=3)
    lengths = [40, 7, 33]
    dec = textgen.TextDecoder(shape, w, 3, 64)
    hidden = torch.randn(80, 120, generator=torch.Generator().manual_seed(5)).half()
    logits = dec.prompt(hidden.cuda(), lengths)
    plain = [Plain(dec, w, b) for b in range(3)]
    at, want = 0, []
    for p, n in zip(plain, lengths):
        x = (hidden[at:at + n].float() @ p.w["inp"].T).half().float() + p.w["positions"][:n]
        want.append(p.run(x)[-1])
        at += n
    for step in range(4):
        got, ref = logits.float().cpu(), torch.stack(want)
        rel = ((got - ref).norm() / ref.norm()).item()
        assert rel < 2e-2, f"step {step}: relative L2 {rel}"
        ids = ref.argmax(1).int()
        logits = dec.step(ids.cuda())
        want = [p.run(p.w["tokens"][i][None] + p.w["positions"][n + step][None])[-1]
                for p, i, n in zip(plain, ids.long(), lengths)]
    torch.cuda.synchronize()
    assert native.ppocr_b200_device_error() == 0
    assert dec.lengths.tolist() == [n + 4 for n in lengths]


def test_generate_is_reproducible_and_bounded(native, cuda):
    from ppocr_b200 import textgen

    shape = textgen.DecoderShape(inputs=120, vocab=18385)
    w = textgen.DecoderWeights(shape, cuda, positions=64, seed=1)
    hidden = torch.randn(50, 120, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2)).half()
    uniform = torch.rand(9, 2, device=cuda, generator=torch.Generator(device=cuda).manual_seed(3))
    full = lambda v: torch.full((2,), v, device=cuda)  # noqa: E731
    runs = []
    for _ in range(2):
        dec = textgen.TextDecoder(shape, w, 2, 64)
        runs.append(dec.generate(hidden, [31, 19], 9, uniform, temperature=full(0.9), top_k=full(40).int(), top_p=full(0.9)))
    torch.cuda.synchronize()
    assert native.ppocr_b200_device_error() == 0
    (ids, probs), (ids2, probs2) = runs
    assert torch.equal(ids, ids2) and torch.equal(probs, probs2)
    assert ((ids >= 0) & (ids < 18385)).all() and ((probs > 0) & (probs <= 1)).all()
    with pytest.raises(ValueError, match="exceed"):
        dec.generate(hidden, [31, 19], 64, uniform)
    with pytest.raises(ValueError, match="hidden"):
        dec.prompt(hidden, [31, 20])
    assert math.isfinite(float(probs.sum()))


def test_example_command(native, cuda, capsys, monkeypatch):
    from ppocr_b200 import textgen

    monkeypatch.setattr("sys.argv", ["textgen", "--lines", "2", "--tokens", "4"])
    textgen.main()
    out = capsys.readouterr().out
    assert "line 0: ids [" in out and "line 1: ids [" in out
