"""Serving the decoder from a cache of pages: prompts in a padded batch, steps of a batch, forks and ends between them, against the decoder
with one dense cache per sequence. The same program runs on the oracle here and on the GPU."""
import numpy as np
import pytest

import b200
from b200.pages import PagedCache
from b200.shlo import programs
from oracle import interp, operators

SHAPE = dict(vocab=97, dim=32, layers=2, heads=4, head_dim=16, hidden=48)


class OracleClient:
    """The calls that serving makes of a client, on NumPy arrays."""

    def compile(self, text):
        client = self

        class Executable:
            def execute(self, args):
                return [np.asarray(a) for a in interp.run_text(text, [a.array if isinstance(a, Held) else a for a in args], wide=True)] if args else [Held(np.zeros(client.shape, np.float32))]
        return Executable()

    def buffer_from_host(self, a, dtype=None):
        return a

    def write_pages(self, cache, rows, slots):
        cache.array = operators.write_pages(cache.array, rows, b200._indices(slots, 1).tolist())

    def copy_pages(self, cache, pairs):
        cache.array = operators.copy_pages(cache.array, b200._indices(pairs, 2).tolist())


class Held:
    def __init__(self, array):
        self.array = array


def weights(dtype):
    return [interp.round_bf16(w) if dtype == "bf16" else w for w in programs.gemma_weights([(n, s) for n, s in programs.gemma_param_spec(**SHAPE)], seed=3)]


def serve(client, dtype, prompts, steps, window=0, sinks=0, pages=24, page_size=4, fork_at=None):
    """Greedy tokens and log probabilities of each prompt, and, from step `fork_at` on, of a fork of the first sequence."""
    def host(x):
        return x.to_numpy() if hasattr(x, "to_numpy") else np.asarray(x)

    W = [client.buffer_from_host(w, dtype="bf16" if dtype == "bf16" else None) for w in weights(dtype)]
    B, T = len(prompts), max(len(p) for p in prompts)
    padded, lengths = np.zeros((B, T), np.int32), np.array([len(p) for p in prompts], np.int32)
    for row, p in zip(padded, prompts):
        row[:len(p)] = p
    kw = dict(SHAPE, dtype=dtype, window=window, sinks=sinks)
    if isinstance(client, OracleClient):
        client.shape = (SHAPE["layers"], 2, pages, page_size, 1, SHAPE["head_dim"])
    prefill = client.compile(programs.gemma_paged_prefill(batch=B, prompt_len=T, **kw).text)
    cache = PagedCache(client, SHAPE["layers"], pages, page_size, 1, SHAPE["head_dim"], dtype)
    seqs = [cache.add() for _ in prompts]
    tok, lp, _, rows = prefill.execute(W + [client.buffer_from_host(padded), client.buffer_from_host(lengths)])
    given, slots, at = cache.extend(seqs, lengths), np.full((B, T), -1, np.int32), 0
    for b, n in enumerate(lengths):
        slots[b, :n] = given[at:at + n]
        at += n
    cache.write(rows, slots.reshape(-1))
    out = {s: ([int(t)], [float(p)]) for s, t, p in zip(seqs, host(tok), host(lp))}
    programs_of = {}
    for i in range(steps):
        if i == fork_at:
            new = cache.fork(seqs[0])
            out[new] = (list(out[seqs[0]][0]), list(out[seqs[0]][1]))
            out[new][0][-1] = (out[new][0][-1] + 1) % SHAPE["vocab"]           # the fork goes another way
            seqs.append(new)
            cache.free(seqs.pop(1))                                           # and a sequence ends
            cache.compact()
        n = len(seqs)
        if n not in programs_of:
            programs_of[n] = client.compile(programs.gemma_paged_step(batch=n, pages=pages, page_size=page_size, width=8, **kw).text)
        args = [np.array([out[s][0][-1] for s in seqs], np.int32), cache.table(seqs, 8), cache.lengths(seqs)]
        tok, table, lens = [client.buffer_from_host(a) for a in args]
        tok, lp, _, rows = programs_of[n].execute(W + [tok, cache.buffer, table, lens])
        cache.write(rows, cache.extend(seqs, [1] * n))
        for s, t, p in zip(seqs, host(tok), host(lp)):
            out[s][0].append(int(t))
            out[s][1].append(float(p))
    return out


PROMPTS = [[5, 9, 2, 40, 41, 7, 3], [1], [60, 61, 62, 63, 64, 65, 66, 67, 68]]


def test_pages_give_the_dense_caches_tokens():
    """Without a window: the tokens of the decoder with a dense cache, one sequence after another."""
    out = serve(OracleClient(), "f32", PROMPTS, 5)
    W = weights("f32")
    for s, prompt in enumerate(PROMPTS):
        kw = dict(SHAPE, dtype="f32", cache_len=len(prompt) + 5)
        tok, _, *caches = interp.run_text(programs.gemma_prefill(prompt_len=len(prompt), **kw).text, W + [np.array(prompt, np.int32)], wide=True)
        ids = interp.run_text(programs.gemma_decode_loop(start=len(prompt), new_tokens=5, **kw).text, W + [tok, *caches], wide=True)[0]
        assert out[s][0] == [int(tok[0]), *ids.tolist()]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (6, 2)])
def test_serving_on_the_gpu(client, window, sinks):
    """In 32 bits: the oracle's tokens and log probabilities, with a fork, an end and a compaction between the steps. (A difference of
    two layers' sums in another order, some 1e-6, against gaps of 1e-3 and more between the best two tokens.)"""
    want = serve(OracleClient(), "f32", PROMPTS, 8, window, sinks, fork_at=3)
    got = serve(client, "f32", PROMPTS, 8, window, sinks, fork_at=3)
    assert want.keys() == got.keys()
    for s in want:
        assert want[s][0] == got[s][0]
        np.testing.assert_allclose(got[s][1], want[s][1], rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
def test_serving_in_16_bits(client):
    """bf16 on the GPU against the oracle on the same weights: the log probability of the first token of each prompt. Its logits come from
    sums of 32 terms of rounded factors, each a 2^-8 of the row's size at the worst; some of them cancel."""
    want, got = (serve(c, "bf16", PROMPTS, 0) for c in (OracleClient(), client))
    for s in want:
        assert abs(want[s][1][0] - got[s][1][0]) < 0.1 * (1 + abs(want[s][1][0]))


def forced(client, dtype, prompts, tokens, pages=24, page_size=4, ahead=0):
    """Log probabilities of the best tokens and entropies of each step [steps + 1, prompts], with `tokens` [steps, prompts] given and not
    chosen. `ahead`: tokens of sequences that come and go in front, so that the pages are others."""
    def host(x):
        return x.to_numpy() if hasattr(x, "to_numpy") else np.asarray(x)

    W = [client.buffer_from_host(w, dtype="bf16" if dtype == "bf16" else None) for w in weights(dtype)]
    B, T = len(prompts), max(len(p) for p in prompts)
    padded, lengths = np.zeros((B, T), np.int32), np.array([len(p) for p in prompts], np.int32)
    for row, p in zip(padded, prompts):
        row[:len(p)] = p
    kw = dict(SHAPE, dtype=dtype)
    if isinstance(client, OracleClient):
        client.shape = (SHAPE["layers"], 2, pages, page_size, 1, SHAPE["head_dim"])
    cache = PagedCache(client, SHAPE["layers"], pages, page_size, 1, SHAPE["head_dim"], dtype)
    seqs = [cache.add() for _ in prompts]
    if ahead:
        others = [cache.add() for _ in range(3)]
        cache.extend(others, [ahead, 1, ahead])
        cache.free(others[1])
    prefill = client.compile(programs.gemma_paged_prefill(batch=B, prompt_len=T, **kw).text)
    step = client.compile(programs.gemma_paged_step(batch=B, pages=pages, page_size=page_size, width=8, **kw).text)
    _, lp, entropy, rows = prefill.execute(W + [client.buffer_from_host(padded), client.buffer_from_host(lengths)])
    given, slots, at = cache.extend(seqs, lengths), np.full((B, T), -1, np.int32), 0
    for b, n in enumerate(lengths):
        slots[b, :n] = given[at:at + n]
        at += n
    cache.write(rows, slots.reshape(-1))
    out = [(host(lp), host(entropy))]
    for tok in tokens:
        args = [client.buffer_from_host(a) for a in (np.asarray(tok, np.int32), cache.table(seqs, 8), cache.lengths(seqs))]
        _, lp, entropy, rows = step.execute(W + [args[0], cache.buffer, *args[1:]])
        cache.write(rows, cache.extend(seqs, [1] * B))
        out.append((host(lp), host(entropy)))
    return np.array(out, np.float64)


@pytest.mark.gpu
def test_steps_in_16_bits(client):
    """bf16, prompts and eight steps with given tokens: the best tokens' log probabilities and the entropies, which change little where two
    tokens change places, against the oracle on the same weights (within what test_serving_in_16_bits allows a log probability), and bit for
    bit the same whichever pages the cache has."""
    tokens = np.random.default_rng(5).integers(0, SHAPE["vocab"], (8, len(PROMPTS)))
    want, got = (forced(c, "bf16", PROMPTS, tokens) for c in (OracleClient(), client))
    assert want.shape == got.shape == (9, 2, len(PROMPTS))
    assert (np.abs(want - got) < 0.1 * (1 + np.abs(want))).all()
    np.testing.assert_array_equal(forced(client, "bf16", PROMPTS, tokens, pages=48, ahead=30), got)


@pytest.mark.gpu
def test_steps_in_32_bits(client):
    tokens = np.random.default_rng(6).integers(0, SHAPE["vocab"], (8, len(PROMPTS)))
    want, got = (forced(c, "f32", PROMPTS, tokens) for c in (OracleClient(), client))
    np.testing.assert_allclose(got, want, rtol=1e-4, atol=1e-5)
