"""The attention operators as a layer uses them: a projection's rows into the cache,
a prompt in one piece and in chunks, then tokens one at a time and with drafts."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import attn_ref as R  # noqa: E402
from attn_cases import ints  # noqa: E402
from r9v_amd import attn, ffi  # noqa: E402

pytestmark = pytest.mark.gpu

KV, GROUP, PAGE, HIDDEN = 2, 4, 16, 256
HEADS = KV * GROUP


class Layer:
    """One layer of an engine: its projections in e4m3, its cache of shuffled pages."""

    def __init__(self, dim, lengths, room, **kw):
        g = torch.Generator().manual_seed(5)
        self.dim, self.kw = dim, kw
        rows = (HEADS + 2 * KV) * dim
        self.w = torch.randn(rows, HIDDEN, generator=g).to(torch.float8_e4m3fn).cuda()
        self.ws = (0.05 + 0.01 * torch.rand(-(-rows // 128), HIDDEN // 128, generator=g)).cuda()
        self.wo = torch.randn(HIDDEN, HEADS * dim, generator=g).to(torch.float8_e4m3fn).cuda()
        self.wos = torch.full((HIDDEN // 128, -(-HEADS * dim // 128)), 0.05).cuda()
        columns = -(-room // PAGE)
        pages = len(lengths) * columns + 3
        self.table = torch.randperm(pages, generator=g)[:len(lengths) * columns].view(len(lengths), columns).int().cuda()
        self.k, self.v = (torch.full((pages, PAGE, KV, dim), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.freqs, self.amplitude = attn.rope_freqs(dim // 2, base=10000.0, scaling="yarn", factor=4.0, original_length=256)

    def slots(self, seq, positions):
        return self.table[seq.long(), (positions // PAGE).long()].long() * PAGE + positions.long() % PAGE

    def turned(self, x, positions, slots):
        """q of the cache's type; k and v in the cache."""
        rows = ffi.matmul_fp8(self.w, self.ws, x, out_dtype=ffi.F32)
        q, k, v = (y.view(x.shape[0], -1, self.dim) for y in rows.split((HEADS * self.dim, KV * self.dim, KV * self.dim), 1))
        q_out = attn.rope_kv(q, k, v, positions, self.freqs, self.k, self.v, slots, amplitude=self.amplitude)
        return (q, k, v), q_out

    def out(self, x, y):
        return ffi.matmul_fp8(self.wo, self.wos, y.reshape(x.shape[0], -1), residual=x.float())

    def check_rows(self, projected, q_out, positions, slots):
        """One rounding to bf16; cosines, sines and products in f32; the angle in f64."""
        at, kk, vv = slots.cpu(), self.k.reshape(-1, KV, self.dim), self.v.reshape(-1, KV, self.dim)
        rot, far = self.dim // 2, float(positions.abs().max())
        for got, x, turns in ((q_out, projected[0], True), (kk[slots], projected[1], True), (vv[slots], projected[2], False)):
            want, size = R.rotated(x, positions, self.freqs, rot, False, self.amplitude)
            if not turns:
                want, size = R.f64(x), 0 * size
            want[..., rot:], size[..., rot:] = R.f64(x)[..., rot:], 0
            tol = 2.0 ** -8 * np.abs(want) * (1 + 2.0 ** -20) + (2.0 ** -21 + 2.0 ** -51 * far) * size + 2.0 ** -25
            assert (np.abs(R.f64(got) - want) <= tol).all()
        assert len(at.unique()) == len(at)

    def check_attention(self, y, q, seq, positions, exact_p):
        """Every row against the definition over the sequence's keys in the cache."""
        got, qq = R.f64(y), R.f64(q)
        for i in seq.unique().tolist():
            rows = (seq == i).nonzero()[:, 0].tolist()
            n = int(positions[rows].max()) + 1
            for kvh in range(KV):
                kk, vv = R.gathered(self.k, self.table[i], n, kvh), R.gathered(self.v, self.table[i], n, kvh)
                for h in range(kvh * GROUP, (kvh + 1) * GROUP):
                    for r in rows:
                        p = int(positions[r])
                        seen = R.intervals(p, n, 0, self.kw.get("window", 0), 0, True)
                        want, size, s = R.attention(qq[r, h], kk, vv, seen, p, self.dim ** -0.5, self.kw.get("softcap", 0.0))
                        assert (np.abs(got[r, h] - want) <= R.bound(want, size, s, self.dim, n, q.dtype, exact_p)).all(), (i, h, p)


@pytest.mark.parametrize("dim,kw", [(64, {}), (128, dict(window=48, softcap=20.0)), (256, {})])
def test_prompts_chunks_tokens_and_drafts(dim, kw):
    prompts, room, new = [70, 1, 133], 200, 4
    layer = Layer(dim, prompts, room, **kw)
    g = torch.Generator().manual_seed(9)
    b = len(prompts)

    def tokens(n):
        return torch.randn(n, HIDDEN, generator=g).to(torch.bfloat16).cuda()

    # the first 32 tokens of each prompt, then the rest onto them
    done = [0] * b
    for last in (32, room):
        now = [min(n, last) - d for n, d in zip(prompts, done)]
        seq = ints([i for i, n in enumerate(now) for _ in range(n)])
        positions = ints([d + j for d, n in zip(done, now) for j in range(n)])
        slots = layer.slots(seq, positions)
        x = tokens(len(seq))
        projected, q = layer.turned(x, positions, slots)
        done = [d + n for d, n in zip(done, now)]
        y = attn.prefill(q, layer.k, layer.v, layer.table, ints(done), ints(np.concatenate(([0], np.cumsum(now))).tolist()), **kw)
        layer.check_rows(projected, q, positions, slots)
        layer.check_attention(y, q, seq, positions, False)
        assert layer.out(x, y).isfinite().all()

    # a token and its drafts, some of them kept: one graph, whose inputs an engine rewrites
    seq = ints([i for i in range(b) for _ in range(new)])
    x, positions = tokens(b * new), ints([0] * (b * new))
    slots, lengths = torch.zeros(b * new, dtype=torch.int64, device="cuda"), ints([0] * b)

    def step():
        projected, q = layer.turned(x, positions, slots)
        y = attn.decode(q.view(b, new, HEADS, dim), layer.k, layer.v, layer.table, lengths, **kw).view(b * new, HEADS, dim)
        return projected, q, y, layer.out(x, y)

    def fill(kept):
        x.copy_(tokens(b * new))
        positions.copy_(ints([d + j for d in kept for j in range(new)]))
        slots.copy_(layer.slots(seq, positions))
        lengths.copy_(ints([d + new for d in kept]))

    fill(done)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        projected, q, y, z = step()
    for kept in ([1, 4, 2], [4, 1, 3], [1, 1, 1]):
        fill(done)
        graph.replay()
        layer.check_rows(projected, q, positions, slots)
        layer.check_attention(y, q, seq, positions, True)
        again = step()
        assert all(torch.equal(a, c) for a, c in zip((q, y, z), again[1:]))
        # a draft that was not kept stands behind the next step's first tokens until it is overwritten
        done = [d + n for d, n in zip(done, kept)]


def test_two_streams_at_once():
    """Calls beside each other, each with memory of its stream, on one cache that both read."""
    lengths, new = [3000, 40, 1700], 2
    layer = Layer(128, lengths, 3000)
    g = torch.Generator().manual_seed(11)
    for c in (layer.k, layer.v):
        c.copy_(torch.randn(c.shape, generator=g))
    q = torch.randn(3, new, HEADS, 128, generator=g).to(torch.bfloat16).cuda()
    p = torch.randn(90, HEADS, 128, generator=g).to(torch.bfloat16).cuda()
    n, off = ints(lengths), ints([0, 50, 60, 90])

    def calls(stream):
        return [attn.decode(q, layer.k, layer.v, layer.table, n, stream=stream), attn.prefill(p, layer.k, layer.v, layer.table, n, off, stream=stream)]

    want = calls(None)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [calls(s) for _ in range(8) for s in streams]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))
