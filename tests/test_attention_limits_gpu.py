"""Attention at the borders of what it accepts: scales and scores near the ends of fp32, weights near the ends of fp16."""
import pytest
import torch

import flashoverlap_b200  # noqa: F401
from attention_oracle import attend, check  # noqa: F401
from flashoverlap_b200 import ops
from test_attention_gpu import BF16, FP16, Paged, check_prompt, ints, randn  # noqa: F401

pytestmark = pytest.mark.gpu

# (batch, sq, sk, heads, kv): so few pairs of tiles that their keys are divided over CTAs, and as many as need no division
SHAPES = [(1, 20, 3000, 8, 1), (2, 300, 300, 4, 2)]


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [1e-30, 1.5e-38, 1e-40])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 3)])
def test_scales_of_almost_nothing(dtype, dim, scale, window, sinks):
    # all scores are nearly zero: a row is the mean of the values it sees, however its keys are divided
    for batch, sq, sk, heads, kv in SHAPES:
        q = randn(batch, sq, heads, dim, dtype=dtype, seed=1)
        k, v = randn(batch, sk, kv, dim, dtype=dtype, seed=2), randn(batch, sk, kv, dim, dtype=dtype, seed=3)
        got = ops.prompt_attention(q, k, v, window=window, sinks=sinks, scale=scale)
        check_prompt(q, k, v, got, window, sinks, scale=scale)
    for lengths in ([40, 300], [9000, 33]):
        p = Paged(lengths, 1, dim, 16, dtype)
        q = randn(len(lengths), 5, dim, dtype=dtype)
        p.check(q, ops.paged_attention(q, p.cache, p.table, p.lengths, window=window, sinks=sinks, scale=scale), window, sinks, scale=scale)


def test_scores_near_the_lowest_number():
    # all scores within 0.8 % of the lowest number of fp32; scaled, they lie between -1357 and -1351
    scale, steps = 4e-36, torch.tensor([2.0 ** 63, 2.0 ** 63 * 255 / 256])
    for batch, sq, sk, heads, kv in SHAPES:
        q = torch.zeros(batch, sq, heads, 64, dtype=BF16, device="cuda")
        k, v = torch.zeros(batch, sk, kv, 64, dtype=BF16, device="cuda"), randn(batch, sk, kv, 64, dtype=BF16, seed=3)
        q[..., 0] = -255 / 128 * 2.0 ** 64
        k[..., 0] = steps[torch.arange(sk) % 7 // 3 % 2].cuda()[None, :, None]
        check_prompt(q, k, v, ops.prompt_attention(q, k, v, scale=scale), scale=scale)


@pytest.mark.parametrize("dim", [64, 128])
def test_small_weights_of_half_precision(dim):
    # Every 16th token has weight 1 and value 0, the others weight 2^-26.5, which is no number of fp16, and value 2^15: the
    # small weights are all of the result.  They are kept with a factor of at least 2^7, next to which an absolute error of
    # 2^-25 is 2^-5.5 of them; then half a step for the weights and half for the result, and the errors of the oracle's bound
    # that are not fp16's (scores of at most 18.4).
    t, big = 18.375, 2.0 ** 15
    delta = 18.4 * (dim + 4) * 2.0 ** -23 + 2.0 ** -21
    for batch, sq, sk, heads, kv in SHAPES + [(1, 1000, 2500, 8, 4)]:
        q, k, v = (torch.zeros(batch, n, h, dim, dtype=FP16, device="cuda") for n, h in ((sq, heads), (sk, kv), (sk, kv)))
        q[..., 0] = 1
        k[:, ::16, :, 0] = t
        v[:], v[:, ::16] = big, 0
        seen = torch.arange(sk - sq + 1, sk + 1, dtype=torch.float64, device="cuda")
        large = torch.ceil(seen / 16)
        small = (seen - large) * torch.exp(torch.tensor(-t, dtype=torch.float64))
        want = big * small / (large + small)
        got = ops.prompt_attention(q, k, v, scale=1.0)
        tol = want * (2.0 ** -5.5 + 2.0 ** -10 + 2 * delta + sk * 2.0 ** -23) + 2.0 ** -25
        assert ((got.double() - want[None, :, None, None]).abs() <= tol[None, :, None, None]).all()
    for lengths in ([200, 17], [6000, 5000]):
        p = Paged(lengths, 1, dim, 16, FP16)
        p.cache.zero_()
        p.cache[:, 0, :, 0, 0] = t
        p.cache[:, 1, :, 1:] = big
        q = torch.zeros(2, 4, dim, dtype=FP16, device="cuda")
        q[..., 0] = 1
        got = ops.paged_attention(q, p.cache, p.table, p.lengths, scale=1.0)
        for s, n in enumerate(lengths):
            large = -(-n // 16)
            small = (n - large) * torch.exp(torch.tensor(-t, dtype=torch.float64)).item()
            want = big * small / (large + small)
            tol = want * (2.0 ** -5.5 + 2.0 ** -10 + 2 * delta + n * 2.0 ** -23) + 2.0 ** -25
            assert (got[s].double() - want).abs().max() <= tol, (n, want, got[s])


def test_what_a_cache_refuses_leaves_no_tokens_behind():
    from flashoverlap_b200.models import PagedKVCache

    with pytest.raises(ValueError, match="float16 or bfloat16"):
        PagedKVCache(4, 16, 2, 64, dtype=torch.float32)
    cache = PagedKVCache(10, 16, 2, 64, dtype=BF16)
    a, b = cache.add(), cache.add()
    x = randn(2, 20, 2, 64, dtype=BF16)
    cache.append([a, b], x, x)
    before = [cache.length(s) for s in (a, b)], [cache.pool.pages(s) for s in (a, b)], cache.pool.free_pages(), cache.data.clone()
    inside = cache.data[0, 0].transpose(0, 1)[None, :14]             # keys that lie in the cache itself
    with pytest.raises(RuntimeError, match="share memory"):
        cache.append([a], inside, inside)
    cache.data.requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        cache.append([b, a], x, x)
    cache.data.requires_grad_(False)
    assert ([cache.length(s) for s in (a, b)], [cache.pool.pages(s) for s in (a, b)], cache.pool.free_pages()) == before[:3]
    assert torch.equal(cache.data, before[3])
    cache.append([b], x[1:], x[1:])                                    # the pages it would have had
    assert cache.length(b) == 40 and cache.pool.free_pages() == before[2] - 1
    cache.free(a)                                                      # pages in front are free now, copies are refused
    pages = cache.pool.pages(b)
    cache.data.requires_grad_()
    for call in (cache.compact, lambda: cache.fork(b)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
    assert cache.pool.pages(b) == pages and cache.pool.num_sequences() == 1 and cache.pool.free_pages() == 7


def test_a_block_that_fails_leaves_no_tokens_behind():
    # the products behind the attention refuse their shapes, or the attention itself does
    from flashoverlap_b200.models import PagedKVCache
    from flashoverlap_b200.models.decoder_block import TPDecoderBlock

    block = TPDecoderBlock(None, 256, 64, 4, 2)
    block._project = lambda h: h @ block.w_qkv.t()
    cache = PagedKVCache(12, 16, 2, 64)
    a, b = cache.add(), cache.add()
    x = randn(1, 20, 2, 64, dtype=BF16)
    cache.append([b], x, x)
    h = randn(40, 256, dtype=BF16)

    def refuse(*args, **kw):
        raise RuntimeError("shape not supported")

    def state():
        return [cache.length(s) for s in (a, b)], [cache.pool.pages(s) for s in (a, b)], cache.pool.free_pages()

    before = state()
    block._after = refuse
    for call in (lambda: block(h, h, 1, 40, cache=cache, seqs=[a]), lambda: block.decode(h[:2], h[:2], cache, [a, b])):
        with pytest.raises(RuntimeError, match="not supported"):
            call()
        assert state() == before
    block._attention = cache.attend = refuse
    block._after = lambda attn, resid: (attn, resid)
    for call in (lambda: block(h, h, 1, 40, cache=cache, seqs=[a]), lambda: block.decode(h[:2], h[:2], cache, [a, b])):
        with pytest.raises(RuntimeError, match="not supported"):
            call()
        assert state() == before
    cache.take_back([b], [5])
    assert cache.length(b) == 15 and cache.pool.free_pages() == before[2] + 1


def test_tangents_are_refused_and_changes_are_counted():
    import torch.autograd.forward_ad as fwAD

    q, k = randn(2, 8, 4, 64, dtype=FP16), randn(2, 16, 2, 64, dtype=FP16)
    cache = randn(6, 2, 2, 8, 64, dtype=FP16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), ints(1, 1)
    with fwAD.dual_level():
        def dual(x):
            return fwAD.make_dual(x, torch.ones_like(x))

        for call in (lambda: ops.prompt_attention(dual(q), k, k), lambda: ops.prompt_attention(q, k, dual(k)),
                     lambda: ops.paged_attention(dual(q[:, 0].contiguous()), cache, table, lens),
                     lambda: ops.paged_attention(q[:, 0], dual(cache), table, lens),
                     lambda: ops.cache_append(dual(k[:, :4].contiguous()), k[:, :4], cache, table, lens),
                     lambda: ops.copy_pages(dual(cache), torch.tensor([[0, 1]]))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):   # tangents do not ask for gradients
                call()
    # what has been saved for a backward pass and is changed here is found out
    for change in (lambda: ops.cache_append(k[:, :4], k[:, :4], cache, table, lens),
                   lambda: ops.copy_pages(cache, torch.tensor([[0, 1]]))):
        w = torch.ones(64, dtype=FP16, device="cuda", requires_grad=True)
        y = (cache * w).sum()
        change()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    out = torch.empty_like(q)
    versions = out._version
    ops.prompt_attention(q, k, k, out=out)
    one = torch.empty_like(q[:, 0])
    ops.paged_attention(q[:, 0], cache, table, lens, out=one)
    assert out._version == versions + 1 and one._version == 1
    with torch.inference_mode():                      # tensors that count nothing
        inf = torch.zeros_like(cache)
        ops.copy_pages(inf, torch.tensor([[0, 1]]))
        ops.cache_append(k[:, :4], k[:, :4], inf, table, lens)
    ops.copy_pages(inf, torch.tensor([[0, 1]]))
