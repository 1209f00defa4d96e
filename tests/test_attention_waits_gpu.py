"""Waits inside the prompt's kernel that run out: what is reported, which rows are NaN, and that later calls are right.
Every launch here is a working one; only the limit of its waits is shorter than the work that they wait for."""
import subprocess
import sys

import pytest
import torch

import flashoverlap_b200  # noqa: F401
from flashoverlap_b200 import ops
from test_attention_gpu import BF16, check_prompt, ints, randn  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def timeout():
    """Sets the limit in ns for one call; the limit and the state are put back."""
    before = ops.attention_set_timeout_ms(10000)

    def limited(ns, call):
        torch.cuda.synchronize()
        ops.attention_set_timeout_ms(ns / 1e6)
        try:
            return call()
        finally:
            torch.cuda.synchronize()
            ops.attention_set_timeout_ms(10000)

    yield limited
    ops.attention_set_timeout_ms(before)
    ops.attention_reset()


# pairs of tiles: fewer than SMs, more (CTAs claim the pairs of others), so few that their keys are divided, padded sequences
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,sq,sk,heads,kv,window,sinks,lengths", [
    (1, 600, 600, 8, 8, 0, 0, None), (2, 2000, 2000, 20, 20, 0, 0, None), (1, 30, 3000, 8, 1, 0, 0, None),
    (3, 1500, 1500, 16, 16, 300, 5, [1500, 0, 700])])
def test_a_wait_that_runs_out(timeout, dim, batch, sq, sk, heads, kv, window, sinks, lengths):
    q = randn(batch, sq, heads, dim, dtype=BF16, seed=1)
    k, v = randn(batch, sk, kv, dim, dtype=BF16, seed=2), randn(batch, sk, kv, dim, dtype=BF16, seed=3)
    lens = None if lengths is None else ints(*lengths)

    def call(out):
        return ops.prompt_attention(q, k, v, window=window, sinks=sinks, lengths=lens, out=out)

    want = call(None)
    check_prompt(q, k, v, want, window, sinks, lengths, heads=(0, heads - 1))
    assert ops.attention_status() == "ok"
    # the shortest limit ends in the first waits, others anywhere or nowhere
    for ns in (0, 300, 600, 1000, 1500, 2000, 3000, 5000, 10000, 100000):
        out = torch.full_like(want, 7.0)
        timeout(ns, lambda: call(out))
        status = ops.attention_status()
        bad = out.isnan().any(-1)
        assert torch.equal(bad, out.isnan().all(-1)), ns                    # whole rows, or none of them
        assert torch.equal(out[~bad], want[~bad]), ns                       # the others are what they should be
        if status == "ok":
            assert ns and not bad.any(), ns
        else:
            assert "ran out" in status and (ns or bad.any())
            with pytest.raises(RuntimeError, match="attention_reset"):
                call(None)
            ops.attention_reset()
            assert ops.attention_status() == "ok"
        assert torch.equal(call(None), want), ns


def test_limits_that_are_refused():
    for ms in (-1, 1e7):
        with pytest.raises(RuntimeError, match="timeout"):
            ops.attention_set_timeout_ms(ms)


def test_a_first_call_that_is_captured():
    # in a process of its own: what the first call sets up is no part of its graph
    code = """
import sys, torch
sys.path.insert(0, %r)
from flashoverlap_b200 import ops
q, k = (torch.randn(1, 300, h, 64, device="cuda", dtype=torch.float16) for h in (4, 2))
out = torch.empty_like(q)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ops.prompt_attention(q, k, k, out=out)
g.replay()
torch.cuda.synchronize()
assert torch.equal(out, ops.prompt_attention(q, k, k)) and ops.attention_status() == "ok"
print("right")
""" % str(__import__("pathlib").Path(__file__).resolve().parents[1])
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "right" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_one_by_one_take_longer_than_a_wait_may(timeout, dim):
    # The last tiles of the first sequence hold a value that is not finite: their rows are computed one by one, 32 a warp over
    # some 4000 tokens, tens of milliseconds, while the other warps wait for the pair that the CTA has claimed.
    batch, n, kv, bad = 8, 4096, 10, 4000
    q, k, v = (randn(batch, n, kv, dim, dtype=BF16, seed=i) for i in range(3))
    clean = ops.prompt_attention(q, k, v)
    check_prompt(q[:1], k[:1], v[:1], clean[:1], heads=(0,))
    v[0, bad, :, 1] = float("inf")
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))

    def call():
        start.record()
        out = ops.prompt_attention(q, k, v)
        end.record()
        return out

    got = timeout(3_000_000, call)
    assert ops.attention_status() == "ok"
    assert start.elapsed_time(end) > 10        # else nothing here has waited for long
    hit = torch.zeros(batch, n, dtype=torch.bool, device="cuda")
    hit[0, bad:] = True
    assert not got[hit][..., 1].isfinite().any()
    assert torch.equal(got[1:], clean[1:]) and torch.equal(got[0, :3840], clean[0, :3840])
    check_prompt(q[:1, :bad], k[:1, :bad], v[:1, :bad], got[:1, :bad], heads=(0, 9))
