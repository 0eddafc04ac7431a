"""Operators that programs name as custom calls, and the bookkeeping of the paged cache: what needs no GPU."""
import re

import numpy as np
import pytest

import b200
from b200.pages import PagedCache
from b200.shlo.builder import Builder
from oracle import interp, operators


def paged_text(B=3, H=8, KH=2, D=64, L=2, P=5, S=16, W=4, dt="bf16", new=True, **kw):
    b = Builder()
    q, cache = b.arg((B, H, D), dt), b.arg((L, 2, P, S, KH, D), dt)
    table, lengths = b.arg((B, W), "i32"), b.arg((B,), "i32")
    n = b.arg((2, B, KH, D), dt) if new else None
    return b.module([b.paged_attention(q, cache, table, lengths, new=n, **kw)])


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_programs_with_operators_compile(dt):
    plan, _ = b200.compile_to_plan(paged_text(dt=dt, layer=1, window=20, sinks=4, scale=0.1))
    assert "operator paged_attention" in plan
    b = Builder()
    q, k, v = b.arg((2, 33, 4, 64), dt), b.arg((2, 33, 2, 64), dt), b.arg((2, 33, 2, 64), dt)
    plan, _ = b200.compile_to_plan(b.module([b.window_attention(q, k, v, window=7)]))
    assert "operator window_attention" in plan
    b = Builder()
    x, t, g = b.arg((5, 1000), dt), b.arg((5,), "i32"), b.arg((5,), "f32")
    lp, *rest = b.token_log_probs(x, t, top=3)
    dx = b.grad(b.reduce_sum(b.mul(lp, g), (0,)), [x])[0]
    assert (dx.shape, dx.dtype) == ((5, 1000), dt)
    plan, _ = b200.compile_to_plan(b.module([lp, *rest, dx]))
    assert "operator token_log_probs " in plan and "operator token_log_probs_grad" in plan


def loss_text(R, V, dt, dependent=False, top=0):
    b = Builder()
    x, t, w = b.arg((R, V), dt), b.arg((R,), "i32"), b.arg((R,), "f32")
    lp, h, n, *best = b.token_log_probs(x, t, top=top)
    # the weights of the log probabilities, scaled behind them in the program; or the entropies, which the call itself gives
    scaled = h if dependent else b.mul(w, b.full((R,), 0.5, "f32"))
    dx = b.grad(b.reduce_sum(b.mul(lp, scaled), (0,)), [x])[0]
    return b.module([b.reduce_sum(b.mul(lp, w), (0,)), dx, n, *best])


def test_loss_and_gradient_become_one_operation():
    def operators_in(*a, **kw):
        plan, _ = b200.compile_to_plan(loss_text(*a, **kw))
        return [w for w in plan.split() if w.startswith("token_log_probs")]
    assert operators_in(300, 5000, "f32") == ["token_log_probs_both"]
    assert operators_in(296, 32760, "f32") == ["token_log_probs_both"] and operators_in(296, 65520, "bf16") == ["token_log_probs_both"]
    two = ["token_log_probs", "token_log_probs_grad"]
    assert operators_in(295, 5000, "f32") == two and operators_in(296, 32761, "f32") == two and operators_in(300, 500, "f32") == two
    assert operators_in(300, 5000, "f32", dependent=True) == two and operators_in(300, 5000, "f32", top=3) == two
    text = loss_text(300, 4100, "f32")
    rng = np.random.default_rng(0)
    args = [rng.standard_normal((300, 4100)).astype(np.float32), rng.integers(-1, 4100, 300).astype(np.int32), rng.standard_normal(300).astype(np.float32)]
    got = interp.run_text(text, args, wide=True)
    np.testing.assert_allclose(got[1], operators.token_log_probs_grad(args[0], args[1], args[2] * 0.5, np.zeros(300), np.zeros(300)), rtol=1e-5, atol=1e-9)


def test_the_assembly_jax_prints():
    # jax.ffi.ffi_call(...)(q, ...): the dictionary stands under one of two names
    for attr in ("backend_config = {layer = 1 : i64, window = 5 : i64}, api_version = 4 : i32", "mhlo.backend_config = {layer = 1 : i64, window = 5 : i64}"):
        text = f"""module @jit_f {{
  func.func public @main(%arg0: tensor<1x2x8xf32>, %arg1: tensor<2x2x3x4x1x8xf32>, %arg2: tensor<1x2xi32>, %arg3: tensor<1xi32>) -> tensor<1x2x8xf32> {{
    %0 = stablehlo.custom_call @b200.paged_attention(%arg0, %arg1, %arg2, %arg3) {{{attr}}} : (tensor<1x2x8xf32>, tensor<2x2x3x4x1x8xf32>, tensor<1x2xi32>, tensor<1xi32>) -> tensor<1x2x8xf32>
    return %0 : tensor<1x2x8xf32>
  }}
}}"""
        plan, _ = b200.compile_to_plan(text)
        assert "operator paged_attention layer=1 window=5" in plan
        rng = np.random.default_rng(0)
        q, c = rng.standard_normal((1, 2, 8)).astype(np.float32), rng.standard_normal((2, 2, 3, 4, 1, 8)).astype(np.float32)
        got = interp.run_text(text, [q, c, np.array([[2, 0]], np.int32), np.array([7], np.int32)])[0]
        np.testing.assert_allclose(got, operators.paged_attention(q, c, np.array([[2, 0]]), [7], layer=1, window=5), rtol=1e-6)


@pytest.mark.parametrize("kw,why", [
    (dict(H=7), "multiple of the number of key-value heads"), (dict(D=60), "multiple of 8"), (dict(D=264), "multiple of 8 from 8 to 256"),
    (dict(layer=2), "layer"), (dict(window=-1), "window"), (dict(sinks=3), "sinks without a window"), (dict(dt="f64"), "f32, bf16 or f16"),
    (dict(W=1 << 26, S=16), "2^30 positions"), (dict(scale=float("inf")), "no number"), (dict(scale=-0.5), "positive"), (dict(scale=0.0), "positive"), (dict(scale=1e300), "positive"), (dict(L=0), "layer"), (dict(S=0), "one position"),
])
def test_paged_attention_refuses(kw, why):
    with pytest.raises(b200.B200Error) as e:
        b200.compile_to_plan(paged_text(**kw))
    assert "b200.paged_attention" in str(e.value) and why in str(e.value)


def refused(target, types, results, config=""):
    names = [f"%arg{i}" for i in range(len(types))]
    text = f"""module @jit_f {{
  func.func public @main({", ".join(f"{n}: tensor<{t}>" for n, t in zip(names, types))}) -> (tensor<{results[0]}>) {{
    %0:{len(results)} = "stablehlo.custom_call"({", ".join(names)}) <{{call_target_name = "{target}", backend_config = {{{config}}}}}> : ({", ".join(f"tensor<{t}>" for t in types)}) -> ({", ".join(f"tensor<{t}>" for t in results)})
    "func.return"(%0#0) : (tensor<{results[0]}>) -> ()
  }}
}}"""
    with pytest.raises(b200.B200Error) as e:
        b200.compile_to_plan(text)
    return str(e.value)


def test_other_refusals():
    paged = ["1x2x8xf32", "1x2x3x4x1x8xf32", "1x2xi32", "1xi32"]
    assert "page table has to be" in refused("b200.paged_attention", [*paged[:2], "2x2xi32", paged[3]], ["1x2x8xf32"])
    assert "lengths" in refused("b200.paged_attention", [*paged[:3], "1xi64"], ["1x2x8xf32"])
    assert "the cache" in refused("b200.paged_attention", [paged[0], "1x2x3x4x1x8xbf16", *paged[2:]], ["1x2x8xf32"])
    assert "the cache" in refused("b200.paged_attention", [paged[0], "1x3x3x4x1x8xf32", *paged[2:]], ["1x2x8xf32"])
    assert "6 dimensions" in refused("b200.paged_attention", [paged[0], "1x2x3x4x8xf32", *paged[2:]], ["1x2x8xf32"])
    assert "new keys" in refused("b200.paged_attention", [*paged, "1x2x1x8xf32"], ["1x2x8xf32"])
    assert "result" in refused("b200.paged_attention", paged, ["1x2x8xbf16"])
    assert "operands" in refused("b200.paged_attention", paged[:3], ["1x2x8xf32"])
    assert "no attribute of this name: softcap" in refused("b200.paged_attention", paged, ["1x2x8xf32"], "softcap = 1 : i64")
    assert "whole number" in refused("b200.paged_attention", paged, ["1x2x8xf32"], "window = 1.5 : f32")
    prompt = ["2x5x4x8xf32", "2x5x2x8xf32", "2x5x2x8xf32"]
    assert "v has to be" in refused("b200.window_attention", [*prompt[:2], "2x5x1x8xf32"], ["2x5x4x8xf32"])
    assert "k has to be" in refused("b200.window_attention", [prompt[0], "2x6x2x8xf32", prompt[2]], ["2x5x4x8xf32"])
    assert "multiple" in refused("b200.window_attention", [prompt[0], "2x5x3x8xf32", "2x5x3x8xf32"], ["2x5x4x8xf32"])
    assert "alternatives" in refused("b200.token_log_probs", ["3x5xf32", "3xi32"], ["3xf32"] * 4 + ["3x6xf32", "3x6xi32"], "top = 6 : i64")
    assert "from 0 to 128" in refused("b200.token_log_probs", ["3x500xf32", "3xi32"], ["3xf32"] * 4 + ["3x129xf32", "3x129xi32"], "top = 129 : i64")
    assert "results" in refused("b200.token_log_probs", ["3x5xf32", "3xi32"], ["3xf32"] * 4, "top = 2 : i64")
    assert "vocabulary is empty" in refused("b200.token_log_probs", ["3x0xf32", "3xi32"], ["3xf32"] * 4)
    assert "tokens" in refused("b200.token_log_probs", ["3x5xf32", "4xi32"], ["3xf32"] * 4)
    assert "not an operator" in refused("b200.decode_attention", paged, ["1x2x8xf32"])


def test_gradient_of_token_log_probs_against_differences():
    rng = np.random.default_rng(3)
    x, t = rng.standard_normal((4, 9)) * 2, np.array([3, -1, 8, 0])
    w = rng.standard_normal((3, 4))
    f = lambda x: sum((a * b).sum() for a, b in zip(operators.token_log_probs(x, t), w))
    dx = operators.token_log_probs_grad(x, t, *w)
    for i in range(4):
        for j in range(9):
            e = np.zeros_like(x)
            e[i, j] = 1e-5
            # central differences: h^2 / 6 times a third derivative of order one, and rounding 1e-16 / h
            assert abs((f(x + e) - f(x - e)) / 2e-5 - dx[i, j]) < 1e-8


class HostClient:
    """Stands in for a client: the cache is a NumPy array of one number per page and position."""

    def __init__(self):
        self.cache = None

    def compile(self, text):
        return self

    def execute(self, args):
        return [None]

    def copy_pages(self, cache, pairs):
        pairs = b200._indices(pairs, 2)
        self.cache = operators.copy_pages(self.cache, pairs.tolist())

    def write_pages(self, cache, rows, slots):
        self.cache = operators.write_pages(self.cache, rows, b200._indices(slots, 1).tolist())


@pytest.mark.parametrize("seed", range(6))
def test_paged_cache_keeps_every_sequence(seed):
    """Random growth, forks, ends and compactions: each sequence reads back the tokens that it was given, pages are never lost."""
    rng = np.random.default_rng(seed)
    size, pages = int(rng.integers(1, 5)), 24
    host = HostClient()
    cache = PagedCache(host, 1, pages, size, 1, 1)
    host.cache = np.zeros((1, 2, pages, size, 1, 1))
    want, token = {}, 1
    for _ in range(300):
        do = rng.integers(0, 10)
        if do < 2 or not want:
            want[cache.add()] = []
        elif do < 6:
            seqs = [s for s in want if rng.random() < 0.6]
            counts = [int(rng.integers(0, 2 * size + 2)) for _ in seqs]
            before = (cache.free_pages, [cache.lengths([s])[0] for s in seqs])
            try:
                slots = cache.extend(seqs, counts)
            except b200.B200Error as e:
                assert e.code == b200.RESOURCE_EXHAUSTED and before == (cache.free_pages, [cache.lengths([s])[0] for s in seqs])
                continue
            values = np.arange(token, token + len(slots), dtype=np.float64)
            token += len(slots)
            cache.write(values.reshape(1, 1, -1, 1, 1).repeat(2, 1), slots)
            for s, n in zip(seqs, counts):
                want[s] += values[:n].tolist()
                values = values[n:]
        elif do < 8:
            s = list(want)[rng.integers(len(want))]
            want[cache.fork(s)] = list(want[s])
        elif do == 8:
            s = list(want)[rng.integers(len(want))]
            cache.free(s)
            del want[s]
        else:
            cache.compact()
            used = {p for s in want for p in cache.table([s])[0]}
            assert used == set(range(len(used)))
        for s, values in want.items():
            table, n = cache.table([s], width=pages)[0], cache.lengths([s])[0]
            assert n == len(values)
            at = np.arange(n)
            assert host.cache[0, 1, table[at // size], at % size, 0, 0].tolist() == values
        assert cache.free_pages == pages - len({p for s in want for p in cache.table([s])[0]})


def test_paged_cache_refuses():
    host = HostClient()
    cache = PagedCache(host, 1, 4, 2, 1, 1)
    host.cache = np.zeros((1, 2, 4, 2, 1, 1))
    s = cache.add()
    for bad in (lambda: cache.extend([s, s], [1, 1]), lambda: cache.extend([s], [-1]), lambda: cache.extend([s], [1, 2]), lambda: cache.free(99),
                lambda: cache.extend([99], [1]), lambda: PagedCache(host, 1, 0, 2, 1, 1), lambda: cache.lengths([5])):
        with pytest.raises(b200.B200Error):
            bad()
    cache.extend([s], [5])
    with pytest.raises(b200.B200Error):
        cache.table([s], width=2)
    with pytest.raises(b200.B200Error):
        cache.extend([s], [4])
    assert cache.free_pages == 1 and cache.lengths([s]).tolist() == [5]


@pytest.mark.parametrize("values,ndim", [([[1, 2]], 1), ([1, 2], 2), ([[1, 2, 3]], 2), ([0.5], 1), ([2**31], 1), ([True], 1)])
def test_indices_are_whole_numbers_of_32_bits(values, ndim):
    with pytest.raises(b200.B200Error):
        b200._indices(values, ndim)


@pytest.mark.parametrize("value", ["0x7F800000 : f32", "0x3F000000 : f32", "nan : f32", "\"large\"", "1.0e+99 : f64"])
def test_scales_that_are_no_numbers(value):
    text = paged_text(scale=0.5)
    assert "scale = 5.000000000e-01 : f32" in text
    with pytest.raises(b200.B200Error, match="scale"):
        b200.compile_to_plan(text.replace("5.000000000e-01 : f32", value))


def test_what_has_no_gradient_says_so():
    b = Builder()
    q, k = b.arg((1, 4, 2, 64), "f32"), b.arg((1, 4, 2, 64), "f32")
    loss = b.reduce_sum(b.window_attention(b.mul(q, q), k, k), (0, 1, 2, 3))
    with pytest.raises(NotImplementedError, match="window_attention"):
        b.grad(loss, [q])
    b = Builder()
    x, t = b.arg((5, 100), "f32"), b.arg((5,), "i32")
    values = b.token_log_probs(x, t, top=2)[3]
    with pytest.raises(NotImplementedError, match="alternatives"):
        b.grad(b.reduce_sum(values, (0, 1)), [x])
    b = Builder()
    x, y = b.arg((1, 4, 2, 64), "f32"), b.arg((1, 4, 2, 64), "f32")
    s = b.stop_gradient(x)
    loss = b.reduce_sum(b.mul(y, b.window_attention(s, s, s)), (0, 1, 2, 3))
    assert b.grad(loss, [y])[0].shape == y.shape


def joined_text(R=300, V=5000, dt="f32", probs=None, grad=None, config="", top=""):
    """A loss and its gradient as the assembly writes them, `probs` and `grad` the types that they claim to give."""
    x, r = f"tensor<{R}x{V}x{dt}>", f"tensor<{R}xf32>"
    probs, grad = [f"tensor<{t}>" for t in probs or [f"{R}xf32"] * 4], f"tensor<{grad or f'{R}x{V}x{dt}'}>"
    return f"""module @jit_f {{
  func.func public @main(%x: {x}, %t: tensor<{R}xi32>, %g: {r}) -> ({probs[0]}, {grad}) {{
    %p:4 = "stablehlo.custom_call"(%x, %t) <{{call_target_name = "b200.token_log_probs", backend_config = {{{top}}}}}> : ({x}, tensor<{R}xi32>) -> ({", ".join(probs)})
    %d = "stablehlo.custom_call"(%x, %t, %p#2, %p#3, %p#1, %g, %g, %g) <{{call_target_name = "b200.token_log_probs_grad", backend_config = {{{config}}}}}> : ({x}, tensor<{R}xi32>, {probs[2]}, {probs[3]}, {probs[1]}, {r}, {r}, {r}) -> {grad}
    "func.return"(%p#0, %d) : ({probs[0]}, {grad}) -> ()
  }}
}}"""


@pytest.mark.parametrize("R,joined", [(300, True), (200, False)])
@pytest.mark.parametrize("kw,why", [
    (dict(grad="2x2xbf16"), "result"), (dict(grad="{R}x5000xbf16"), "result"), (dict(grad="{R}x4999xf32"), "result"), (dict(probs=["3xf32"] + ["{R}xf32"] * 3), "result"),
    (dict(probs=["{R}xf32"] * 3 + ["{R}xf64"]), "result"), (dict(config="top = 0 : i64"), "no attribute"), (dict(config="scale = 1.0 : f32"), "no attribute"),
    (dict(top="top = 3 : i64"), "results"), (dict(top="scale = 1.0 : f32"), "no attribute")])
def test_a_loss_with_its_gradient_refuses_what_either_would(R, joined, kw, why):
    """Also in rows that both are made of by one kernel, which writes results of the sizes that the logits give."""
    plan, _ = b200.compile_to_plan(joined_text(R))
    assert ("token_log_probs_both" in plan) == joined
    kw = {k: [t.format(R=R) for t in v] if isinstance(v, list) else v.format(R=R) for k, v in kw.items()}
    with pytest.raises(b200.B200Error, match=why):
        b200.compile_to_plan(joined_text(R, **kw))


@pytest.mark.parametrize("R", [1, 2, 3, 8, 300])
@pytest.mark.parametrize("V,top", [(300000, 128), (600000, 64), (1000000, 128), (2000000, 64)])
def test_alternatives_of_few_rows_of_large_vocabularies(R, V, top):
    """What is taken of many rows is taken of one: few rows are cut into more parts only as far as their alternatives can be joined."""
    b = Builder()
    x, t = b.arg((R, V), "bf16"), b.arg((R,), "i32")
    plan, _ = b200.compile_to_plan(b.module(b.token_log_probs(x, t, top=top)))
    assert "operator token_log_probs top" in plan


@pytest.mark.parametrize("R", [1, 300])
def test_more_alternatives_than_can_be_joined(R):
    b = Builder()
    x, t = b.arg((R, 1200000), "bf16"), b.arg((R,), "i32")
    with pytest.raises(b200.B200Error, match="more alternatives"):
        b200.compile_to_plan(b.module(b.token_log_probs(x, t, top=128)))


@pytest.mark.parametrize("generic", [False, True])
@pytest.mark.parametrize("operands,results,fine", [
    ("dense<[2, 1, 0]> : tensor<3xindex>, dense<[5, 4, 3, 2, 1, 0]> : tensor<6xindex>, dense<[1, 0]> : tensor<2xindex>, dense<0> : tensor<1xindex>", "dense<[2, 1, 0]> : tensor<3xindex>", True),
    ("dense<[2, 1, 0]> : tensor<3xindex>, dense<[5, 4, 3, 2, 1, 0]> : tensor<6xindex>, dense<[0, 1]> : tensor<2xindex>, dense<0> : tensor<1xindex>", "dense<[2, 1, 0]> : tensor<3xindex>", False),
    ("dense<[2, 1, 0]> : tensor<3xindex>, dense<[5, 4, 3, 2, 1, 0]> : tensor<6xindex>, dense<[1, 0]> : tensor<2xindex>, dense<0> : tensor<1xindex>", "dense<[1, 2, 0]> : tensor<3xindex>", False),
    ("dense<[2, 1, 0]> : tensor<3xindex>, dense<[5, 4, 3, 2, 1, 0]> : tensor<6xindex>, dense<[1, 0]> : tensor<2xindex>", "dense<[2, 1, 0]> : tensor<3xindex>", False),
    ("dense<[2, 1, 0]> : tensor<3xindex>, dense<[4, 5, 3, 2, 1, 0]> : tensor<6xindex>, dense<[1, 0]> : tensor<2xindex>, dense<0> : tensor<1xindex>", "dense<[2, 1, 0]> : tensor<3xindex>", False),
    ("dense<[2, 1, 0]> : tensor<3xindex>, dense<[4, 3, 2, 1, 0]> : tensor<5xindex>, dense<[1, 0]> : tensor<2xindex>, dense<0> : tensor<1xindex>", "dense<[2, 1, 0]> : tensor<3xindex>", False),
])
def test_layouts_are_row_major(operands, results, fine, generic):
    """jax.ffi.ffi_call writes a layout for each operand and result; any but row-major is refused, not read in the wrong order."""
    types = ["tensor<1x2x8xf32>", "tensor<2x2x3x4x1x8xf32>", "tensor<1x2xi32>", "tensor<1xi32>"]
    attrs = f"api_version = 4 : i32, operand_layouts = [{operands}], result_layouts = [{results}]"
    call = (f'"stablehlo.custom_call"(%arg0, %arg1, %arg2, %arg3) <{{call_target_name = "b200.paged_attention", {attrs}}}>' if generic else
            f"stablehlo.custom_call @b200.paged_attention(%arg0, %arg1, %arg2, %arg3) {{{attrs}}}")
    text = f"""module @jit_f {{
  func.func public @main({", ".join(f"%arg{i}: {t}" for i, t in enumerate(types))}) -> tensor<1x2x8xf32> {{
    %0 = {call} : ({", ".join(types)}) -> tensor<1x2x8xf32>
    return %0 : tensor<1x2x8xf32>
  }}
}}"""
    if fine:
        assert "operator paged_attention" in b200.compile_to_plan(text)[0]
    else:
        with pytest.raises(b200.B200Error, match="b200.paged_attention.*layout"):
            b200.compile_to_plan(text)


@pytest.mark.parametrize("config", ['"{window = 5 : i64}"', '"\\7B\\22window\\22: 5}"', '"window=5"'])
def test_a_configuration_in_a_string_is_refused(config):
    """Attributes that would not be read; a call of the earlier form without any is fine."""
    text = paged_text(window=5)
    given = re.sub(r"backend_config = \{[^}]*\}", lambda m: f"backend_config = {config}", text)
    assert given != text
    with pytest.raises(b200.B200Error, match="b200.paged_attention.*backend_config"):
        b200.compile_to_plan(given)
    plain = re.sub(r"backend_config = \{[^}]*\}", 'backend_config = ""', text).replace("api_version = 4", "api_version = 2")
    assert "operator paged_attention" in b200.compile_to_plan(plain)[0]
