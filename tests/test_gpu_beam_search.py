"""GPU: Decoder.beam_search, which runs the beam selection and the paged cache
together, against the same search with the cache and the selection restated in 64
bits (paged_ref.py) around the decoder's own steps; and a loop of selection,
reordering, growth, new rows and attention, as a server with several requests
runs it."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import layout as lay_mod, ops, paged, synth_gpu  # noqa: E402
from fleet_moe.layout import DSV2_LITE  # noqa: E402

V, N_LAYERS, MAX_POS = 102400, 3, 200


def say(msg: str) -> None:
    print(f"[gpu] {msg}", flush=True)


@pytest.fixture(scope="module")
def decoder():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    lay = lay_mod.model_layout(DSV2_LITE, n_layers=N_LAYERS)
    blob = torch.empty(lay.nbytes, dtype=torch.uint8, device="cuda")
    synth_gpu.fill_model(blob, lay, seed=0)
    return ops.Decoder(blob, lay, DSV2_LITE, max_pos=MAX_POS)


def prompt_of(n: int, seed: int = 3) -> torch.Tensor:
    return torch.from_numpy(np.random.default_rng(seed).integers(0, V, n).astype(np.int32)).cuda()


def restated(dec, prompt, n_beams, n_steps, eos):
    """The search with ref.Cache and ref.beam_select; the prompt and the single
    steps are the decoder's."""
    n = prompt.numel()
    cache = ref.Cache(40, n_beams, 4, N_LAYERS)
    dec.prefill(prompt)
    cache.grow([n] + [0] * (n_beams - 1))
    cache.append(ref.values(dec.cache[:, :n].cpu().numpy()), [0] + [n] * n_beams)
    cache.remap([0] * n_beams)
    row = torch.zeros(V, device="cuda")
    dec.attn.lm_head_into(dec.x, dec._addr("final_norm"), dec._addr("lm_head"), row, dec.token_out)
    logits = np.zeros((1, n_beams, V), np.float32)
    logits[0, 0] = row.cpu().numpy()
    scores = np.full((1, n_beams), -np.inf, np.float32)
    scores[0, 0] = 0
    finished = np.zeros((1, n_beams), bool)
    found = np.zeros((n_beams, n_steps), np.int64)
    for step in range(n_steps):
        at = n + step - 1
        if step:
            new = np.zeros((N_LAYERS, n_beams, ref.ROW), np.float32)
            for b in range(n_beams):
                rows = np.stack([cache.values(b, k) for k in range(N_LAYERS)])
                dec.cache[:, :at].copy_(torch.from_numpy(ref.bits(rows.astype(np.float32))))
                dec.reset(at)
                dec.token.fill_(int(found[b, step - 1]))
                dec.enqueue_step(row, feed_back=False)
                logits[0, b] = row.cpu().numpy()
                new[:, b] = ref.values(dec.cache[:, at].cpu().numpy())
            assert cache.grow([1] * n_beams)
            cache.append(new, list(range(n_beams + 1)))
        best = ref.beam_select(logits, scores, finished, n_beams, eos)[0]
        parents = [r[1] for r in best]
        cache.remap(parents)
        found = found[parents]
        found[:, step] = [r[2] for r in best]
        scores = np.array([[r[0] for r in best]], np.float32)
        finished = np.array([[bool(r[3]) for r in best]])
        if eos >= 0 and finished.all():
            found[:, step:] = eos
            break
    return found, scores[0]


def check(dec, n, n_beams, n_steps, eos=-1):
    say(f"prompt {n} beams {n_beams} steps {n_steps} eos {eos}")
    prompt = prompt_of(n)
    found, scores = dec.beam_search(prompt, n_beams, n_steps, eos)
    want, ws = restated(dec, prompt, n_beams, n_steps, eos)
    assert np.array_equal(found.cpu().numpy(), want)
    # a select rounds a score by half a step and adds a log sum within 2^-20
    tol = n_steps * (2.0**-24 * np.abs(ws).max() + 2.0**-20)
    assert np.abs(scores.cpu().numpy() - ws).max() <= tol
    assert dec.status() == 0
    return found


# a prompt of one token (a step), of a page and a part, an exact page, across a page's end
@pytest.mark.parametrize("n, n_beams, n_steps", [(1, 2, 3), (70, 3, 4), (64, 4, 3), (61, 3, 6),
                                                 (5, 1, 4), (9, 8, 1)])
def test_search(decoder, n, n_beams, n_steps):
    check(decoder, n, n_beams, n_steps)


def test_one_beam_is_the_best_token(decoder):
    """One beam and one step: the greedy pick, from the exact cache."""
    prompt = prompt_of(40)
    found, scores = decoder.beam_search(prompt, 1, 1)
    decoder.prefill(prompt)
    assert int(found[0, 0]) == int(decoder.token_out.item()) and float(scores[0]) < 0


def test_search_ends_at_eos(decoder):
    """The first step's best token as the end: its beam keeps it, the others go on;
    and with one beam the search ends at once."""
    n = 20
    eos = int(decoder.beam_search(prompt_of(n), 1, 1)[0][0, 0])
    found = check(decoder, n, 3, 4, eos).cpu().numpy()
    assert (found == eos).all(axis=1).any() and not (found == eos).all()
    assert (check(decoder, n, 1, 5, eos).cpu().numpy() == eos).all()


def test_refusals(decoder):
    for n, beams, steps in ((0, 2, 1), (5, 0, 1), (5, 65, 1), (5, 2, 0), (100, 2, MAX_POS - 98)):
        with pytest.raises(ValueError):
            decoder.beam_search(prompt_of(n), beams, steps)
    with pytest.raises(ValueError):
        decoder.beam_search(prompt_of(4), 2, 2, eos=V)
    check(decoder, 100, 1, 2)


@pytest.mark.parametrize("seed", [0, 1])
def test_a_server_of_beams(seed):
    """Three requests of four beams: every step selects, moves the states to the chosen
    parents, makes room, writes the new rows of two layers and attends, on the device
    and restated."""
    rng = np.random.default_rng(seed)
    groups, beams, vocab, heads = 3, 4, 500, 16
    n = groups * beams
    dev = paged.PagedCache.empty(60, n, 6, 2)
    want = ref.Cache(60, n, 6, 2)
    select = ops.BeamSelector(groups, beams, vocab=vocab, eos=7)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lens = [int(rng.integers(1, 140)) if s % beams == 0 else 0 for s in range(n)]
    at = np.concatenate([[0], np.cumsum(lens)])
    rows = ref.bf16(rng.normal(size=(2, sum(lens), ref.ROW)))
    heirs = [s // beams * beams for s in range(n)]
    assert want.grow(lens)
    want.append(rows, at)
    want.remap(heirs)
    dev.grow(i32(lens))
    dev.append(torch.from_numpy(ref.bits(rows)).cuda(), i32(at))
    dev.remap(i32(heirs))
    scores = torch.full((groups, beams), -np.inf, device="cuda")
    scores[:, 0] = 0
    done = torch.zeros((groups, beams), dtype=torch.uint8, device="cuda")
    for step in range(6):
        say(f"seed {seed} step {step}")
        logits = ref.bf16(rng.normal(size=(groups, beams, vocab)) * 2)
        best = ref.beam_select(logits, scores.cpu().numpy(), done.cpu().numpy().astype(bool), beams, 7)
        got = select.select(torch.from_numpy(logits).cuda().view(n, vocab), scores, done)
        for g in range(groups):
            assert got["parents"][g].tolist() == [r[1] for r in best[g]]
            assert got["tokens"][g].tolist() == [r[2] for r in best[g]]
        scores, done = got["scores"], got["finished"]
        dev.remap(got["parents"].reshape(n))
        want.remap([r[1] for rows in best for r in rows])
        assert want.grow([1] * n)
        dev.grow(i32([1] * n))
        rows = ref.bf16(rng.normal(size=(2, n, ref.ROW)))
        want.append(rows, list(range(n + 1)))
        dev.append(torch.from_numpy(ref.bits(rows)).cuda())
        q = ref.bf16(rng.normal(size=(n, heads, ref.ROW)) * 0.5)
        for layer in range(2):
            out, lse = dev.attend(torch.from_numpy(ref.bits(q)).cuda(), layer=layer)
            out, lse = ref.values(out.cpu().numpy()), lse.cpu().numpy()
            for s in range(n):
                o, e, to, te = ref.attend(want.values(s, layer), q[s:s + 1], [want.lens[s] - 1],
                                          paged.SOFTMAX_SCALE)
                assert (np.abs(out[s] - o[0]) <= to[0]).all()
                assert (np.abs(lse[s] - e[0]) <= te[0]).all()
    torch.cuda.synchronize()
    assert dev.status() == 0
    assert np.array_equal(dev.table.cpu().numpy(), want.table())
    used = want.compact()
    assert int(dev.compact().item()) == used
    assert np.array_equal(dev.table.cpu().numpy(), want.table())


def test_search_up_to_the_last_position(decoder):
    check(decoder, MAX_POS - 3, 2, 4)


def test_search_of_a_decoder_with_separate_launches(decoder):
    """The same tokens and scores, also where steps are replayed from a graph, and from
    a prompt on the host or in 64 bits."""
    want = decoder.beam_search(prompt_of(30), 3, 4)
    other = ops.Decoder(decoder.blob, decoder.layout, DSV2_LITE, max_pos=MAX_POS, fused=False)
    for p in (prompt_of(30), prompt_of(30).cpu(), prompt_of(30).long()):
        got = other.beam_search(p, 3, 4)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    other.capture()
    got = other.beam_search(prompt_of(30), 3, 4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert other.status() == 0
