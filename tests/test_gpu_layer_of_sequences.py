"""GPU: the calls around a layer's matrix products together, as a server steps several
sequences through it: norm, projection, queries rotated, projected rows into the pages,
attention over shared pages, residual with the next norm, and the experts; eagerly and as a
captured graph, and against the batch-1 decoder's own layer."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import ops, paged, rope, synth  # noqa: E402
from fleet_moe.layout import DSV2_LITE  # noqa: E402

HEADS, NOPE, ROPE, LORA, V = 16, 128, 64, 512, 128
HIDDEN = DSV2_LITE.hidden


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def bits(t):
    return t.to(torch.bfloat16).view(torch.int16)


def wide(t):
    return t.view(torch.bfloat16).float()


class Layer:
    """One layer's weights, N(0, 0.02^2) as the model's, and its products in plain torch."""

    def __init__(self, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        w = lambda *s: 0.02 * torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.norm_in = bits(1 + w(HIDDEN))
        self.norm_post = bits(1 + w(HIDDEN))
        self.kv_norm = bits(1 + w(LORA))
        self.qkv = w(HEADS * (NOPE + ROPE) + LORA + ROPE, HIDDEN).bfloat16().float()
        kv_b = w(HEADS, NOPE + V, LORA).bfloat16().float()
        self.uk, self.uv = kv_b[:, :NOPE].contiguous(), kv_b[:, NOPE:].transpose(1, 2).contiguous()
        self.o = w(HIDDEN, HEADS * V).bfloat16().float()

    def project(self, h, q):
        """The fused projection's rows; the absorbed queries' first part into q."""
        row = (wide(h) @ self.qkv.T).bfloat16()
        heads = row[:, : HEADS * (NOPE + ROPE)].view(-1, HEADS, NOPE + ROPE)
        nope = heads[..., :NOPE].float().transpose(0, 1).contiguous()
        q[..., :LORA].copy_(torch.bmm(nope, self.uk).transpose(0, 1).bfloat16().view(torch.int16))
        return row.view(torch.int16)

    def outward(self, o):
        v = torch.bmm(wide(o).transpose(0, 1).contiguous(), self.uv).transpose(0, 1)
        return bits(v.bfloat16().float().reshape(-1, HEADS * V) @ self.o.T)


class Server:
    """Sequences of a request's beams over one layer."""

    def __init__(self, n_seqs, groups, tokens):
        self.w = Layer(1)
        blob, lay = synth.moe_layer_blob(seed=0, layer=1, dims=DSV2_LITE)
        self.experts = ops.DeviceLayer.from_host(blob, lay, 1, DSV2_LITE)
        self.runner = ops.GroupedRunner(tokens)
        self.cache = paged.PagedCache.empty(60, n_seqs, 20, 1)
        self.cache.pool.fill_(0xFF)
        self.shared = paged.SharedPrefix(self.cache, i32(groups), tokens, HEADS)
        self.rope = ops.Rotary(rope.frequencies(), rope.magnitude())
        self.h_f32 = torch.empty((tokens, HIDDEN), device="cuda")

    def step(self, x, start=None, keep=None):
        """x int16 [n][2048] through the layer, its positions already grown."""
        n, w = x.shape[0], self.w
        _, h = ops.residual_norm(x, norm=w.norm_in)
        q = torch.empty((n, HEADS, LORA + ROPE), dtype=torch.int16, device="cuda")
        row = w.project(h, q)
        pe = row[:, : HEADS * (NOPE + ROPE)].view(n, HEADS, NOPE + ROPE)[..., NOPE:]
        self.cache.rotate(self.rope, pe, start, out=q[..., LORA:])
        self.cache.append_latent(row[:, HEADS * (NOPE + ROPE):], self.rope, w.kv_norm, start)
        o, lse = self.shared.attend(q, start)
        y = w.outward(o)
        x1, h1 = ops.residual_norm(x, y, w.norm_post, h_f32=self.h_f32[:n])
        m = ops.moe(self.experts, self.h_f32[:n], self.runner)["out"]
        x2, h2 = ops.residual_norm(x1, m, w.norm_in)
        if keep is not None:
            keep.update(h=h, row=row, q=q, o=o, lse=lse, y=y, x1=x1, h1=h1, m=m, x2=x2, h2=h2)
        return x2


def host(t):
    return ref.values(t.cpu().contiguous().numpy()).astype(np.float64)


def near(got, want, rel, size):
    d = np.abs(got - want)
    assert (d <= rel * np.abs(want) + size).all(), np.nanmax(d - rel * np.abs(want) - size)


def test_a_step_of_beams_stage_by_stage():
    """A prompt, its beams, and steps of them; every stage from the stage before as it came
    out, in 64 bits. (Tolerances: half a step of bf16, 2^-8, and 2^-17 of the sizes for the
    sums in fp32; the pages' 8 bits enter by reading them back.)"""
    rng = np.random.default_rng(3)
    s = Server(4, [0, 3, 4], 250)
    x = torch.from_numpy(ref.bits(ref.bf16(rng.normal(size=(250, HIDDEN))))).cuda()
    s.cache.grow(i32([160, 0, 0, 90]))
    start = i32([0, 160, 160, 160, 250])
    keep = {}
    s.step(x, start, keep)                          # nothing shared yet: never updated
    for step in range(3):
        s.cache.remap(i32([0, 0, 0, 3] if step == 0 else [1, 2, 0, 3]))
        lens = [160 + step] * 3 + [90 + step]
        assert s.shared.update().tolist() == [2, 0]
        s.cache.grow(i32([1, 1, 1, 1]))
        x = torch.from_numpy(ref.bits(ref.bf16(rng.normal(size=(4, HIDDEN))))).cuda()
        s.step(x, None, keep)
    assert s.cache.status() == 0
    lens = [n + 1 for n in lens]
    k = {n: (t.cpu().numpy() if n == "lse" else host(t)) for n, t in keep.items()}
    xs = host(x)
    unit = lambda v: v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6)  # noqa: E731
    w = s.w
    near(k["h"], unit(xs) * host(w.norm_in), 2.0**-8 + 2.0**-17, 0)
    # the rotated part of the queries
    pos = np.array(lens) - 1
    ang = pos[:, None] * rope.frequencies().astype(np.float64)
    co, si = np.cos(ang)[:, None], np.sin(ang)[:, None]
    pe = k["row"][:, : HEADS * 192].reshape(4, HEADS, 192)[..., 128:]
    a, b = pe[..., 0::2], pe[..., 1::2]
    near(k["q"][..., 512:], np.concatenate([a * co - b * si, b * co + a * si], -1), 2.0**-8,
         2.0**-19 * np.abs(pe).max())
    # the rows that the pages hold of the newest positions, and the attention over all of them
    rows = torch.zeros((sum(lens), 576), dtype=torch.int16, device="cuda")
    s.cache.read(rows, i32(np.concatenate([[0], np.cumsum(lens)])))
    held, at = host(rows), 0
    for i, n in enumerate(lens):
        c = k["row"][i, HEADS * 192: HEADS * 192 + 512]
        new = held[at + n - 1]
        want = unit(c) * host(w.kv_norm)
        near(new[:512], want, 2.0**-4, 2.0**-9 * np.abs(held[at: at + n, :512]).max())
        out, lse, tol, tl = ref.attend(held[at: at + n], k["q"][i: i + 1], [n - 1],
                                       paged.SOFTMAX_SCALE)
        assert (np.abs(k["o"][i: i + 1] - out) <= tol).all()
        assert (np.abs(k["lse"][i: i + 1] - lse) <= tl).all()
        at += n
    x1 = xs + k["y"]
    near(k["x1"], x1, 2.0**-8, 0)
    near(k["h1"], unit(x1) * host(w.norm_post), 2.0**-8 + 2.0**-17, 0)
    assert torch.equal(s.h_f32[:4], ops.bf16_bits_to_f32(keep["h1"]))
    near(k["x2"], k["x1"] + k["m"], 2.0**-8, 0)


def test_captured_steps_replayed_between_eager_ones():
    rng = np.random.default_rng(4)
    s = Server(4, [0, 4], 150)
    draw = lambda n: torch.from_numpy(ref.bits(ref.bf16(rng.normal(size=(n, HIDDEN))))).cuda()  # noqa: E731
    s.cache.grow(i32([150, 0, 0, 0]))
    s.step(draw(150), i32([0, 150, 150, 150, 150]))
    s.cache.remap(i32([0, 0, 0, 0]))
    c = s.cache
    state = (c.pool, c.table, c.lens, c.refs)
    saved = [t.clone() for t in state]
    x, out = draw(4), torch.zeros((4, HIDDEN), dtype=torch.int16, device="cuda")
    parents, ones = i32([1, 0, 2, 2]), i32([1] * 4)

    def run():
        c.remap(parents)
        s.shared.update()
        c.grow(ones)
        out.copy_(s.step(x))

    def back():
        for t, v in zip(state, saved):
            t.copy_(v)

    want = []
    for _ in range(2):
        run()
        want.append((out.clone(), c.lens.clone()))
    back()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream), torch.cuda.graph(g, stream=stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    for rep in range(3):
        back()
        for k in range(2):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[k][0]) and torch.equal(c.lens, want[k][1]), (rep, k)
        back()
        run()
        assert torch.equal(out, want[0][0]), rep
    assert c.status() == 0


def test_a_prompt_like_the_decoders_attention():
    """A layer's attention half of a prompt, token by token, beside ops.AttnDecoder's on a bf16
    cache: the difference is what the pages' 8 bits, 2^-4 of a value, leave of sums over them."""
    from fleet_moe import _lib
    rng = np.random.default_rng(5)
    n = 40
    s = Server(1, [0, 1], n)
    w = s.w
    flat = lambda t: t.bfloat16().contiguous().view(torch.int16)  # noqa: E731
    kv_b = torch.cat([w.uk, w.uv.transpose(1, 2)], 1).reshape(HEADS * (NOPE + V), LORA)
    held = [w.norm_in, flat(w.qkv), w.kv_norm, flat(kv_b), flat(w.o)]
    layer = _lib.FleetAttnLayer(*[t.data_ptr() for t in held])
    dec = ops.AttnDecoder()
    cos, sin = (torch.from_numpy(t).cuda() for t in rope.yarn_tables(64))
    cache = torch.zeros((64, 576), dtype=torch.int16, device="cuda")
    x = torch.from_numpy(ref.bits(ref.bf16(rng.normal(size=(n, HIDDEN))))).cuda()
    want = torch.empty((n, HIDDEN), device="cuda")
    for t in range(n):
        dec.attn_into(layer, ops.bf16_bits_to_f32(x[t]), want[t], cache, t, cos=cos, sin=sin)
    s.cache.grow(i32([n]))
    keep = {}
    s.step(x, i32([0, n]), keep)
    assert dec.status() == 0 and s.cache.status() == 0
    got, y = ops.bf16_bits_to_f32(keep["x1"]), want - ops.bf16_bits_to_f32(x)
    # Rounding to 8 bits is off by 2^-4 of a value at most, 2^-4 / sqrt(3) in the mean square: the
    # outputs by no more of their length than that, their scores' share of it again, and the
    # roundings to bf16 (2^-8). A sine of 2^-3, three times as much, is a cosine of 1 - 2^-7.
    g = got - ops.bf16_bits_to_f32(x)
    cosine = (g * y).sum(1) / (g.norm(dim=1) * y.norm(dim=1))
    assert (cosine > 1 - 2.0**-7).all(), cosine.min()
    rows = torch.zeros((n, 576), dtype=torch.int16, device="cuda")
    s.cache.read(rows, i32([0, n]))
    a, b = host(rows), host(cache[:n])
    size = np.abs(b).reshape(-1, 576).max()
    # (half a step of 8 bits, 2^-4; of bf16 at the decoder, 2^-8, and of the projection's rows)
    assert (np.abs(a - b) <= (2.0**-4 + 2.0**-7) * np.abs(b) + 2.0**-9 * size + 2.0**-7 * size).all()
