"""The serving path that runs the paged KV cache operators together: ``chain.layer_step`` against the
same layer computed over the whole sequence, and the beam-decoding example's page bookkeeping."""

import importlib.util
import os

import pytest
import torch

from tests.conftest import REPO

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("paged_decode", os.path.join(REPO, "examples", "paged_decode.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_layer_step_in_chunks_matches_the_whole_sequence():
    """A prompt, a chunk and single tokens through ``layer_step`` give what ``layer_forward`` gives for
    the whole sequence.  The cache rounds keys and values to e4m3 under power-of-two scales: half of
    2^-3 relative for each, a random error that attention averages; the layer output is compared in
    the 2-norm, with 2^-4 (one code's rounding) as the bound."""
    from ntops_b200 import chain, kv_cache

    B, S, page = 2, 150, 16
    dev = "cuda"
    wts = chain.LayerWeights(dev, seed=3)
    sin, cos = chain.rope_tables(S, dev)
    x = torch.randn((B, S, chain.HIDDEN), device=dev).to(torch.bfloat16)
    want = chain.layer_forward(x, wts, sin, cos, fused=False).float()
    cache = kv_cache.PagedKVCache.allocate(1, 2 * B * S // page + 4, chain.KV_HEADS, page, chain.HEAD_DIM)
    refs = torch.zeros(cache.num_pages, dtype=torch.int32, device=dev)
    table = torch.full((B, -(-S // page)), -1, dtype=torch.int32, device=dev)
    got, done = [], 0
    for n in (100, 30, 1, 1, 18):
        start = torch.full((B,), done, dtype=torch.int32, device=dev)
        table, refs, missing = kv_cache.extend(cache, table, refs, start + n)
        assert missing.tolist() == [0]
        got.append(chain.layer_step(x[:, done:done + n], wts, sin, cos, cache.layer(0), table, start, start + n))
        done += n
    got = torch.cat(got, 1).float()
    rel = (got - want).norm() / want.norm()
    assert rel < 2.0**-4, rel
    assert ((got - want).norm(dim=-1) / want.norm(dim=-1)).max() < 2.0**-3


def test_ragged_prompts_leave_other_rows_alone():
    from ntops_b200 import chain, kv_cache

    dev, page = "cuda", 16
    wts = chain.LayerWeights(dev, seed=4)
    sin, cos = chain.rope_tables(64, dev)
    x = torch.randn((2, 40, chain.HIDDEN), device=dev).to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=dev)

    def run(rows, lengths):
        cache = kv_cache.PagedKVCache.allocate(1, 16, chain.KV_HEADS, page, chain.HEAD_DIM)
        table, refs, _ = kv_cache.extend(cache, torch.full((len(rows), 4), -1, **i32), torch.zeros(16, **i32),
                                         torch.tensor(lengths, **i32))
        return chain.layer_step(x[rows], wts, sin, cos, cache.layer(0), table, torch.zeros(len(rows), **i32),
                                torch.tensor(lengths, **i32))

    both = run([0, 1], [40, 23])
    torch.testing.assert_close(both[0], run([0], [40])[0], rtol=0, atol=0)
    torch.testing.assert_close(both[1, :23], run([1], [23])[0, :23], rtol=0, atol=0)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_paged_decode_example(dtype):
    r = _example().decode(layers=1, requests=3, beams=2, prompt=40, steps=10, dtype=dtype)
    assert r["missing"] == 0
    assert r["history"].shape == (3, 2, 10)
    # every reference is accounted for, used pages are at the front, and no entry points past them
    table, refs = r["table"].cpu(), r["refs"].cpu()
    want = torch.bincount(table[table >= 0].long(), minlength=refs.numel()).int()
    assert torch.equal(refs, want)
    assert int((refs > 0).sum()) == r["used"] and int(table.max()) < r["used"] and (refs[r["used"]:] == 0).all()
    need = -(-r["lengths"].cpu() // 16)
    assert torch.equal((table >= 0).sum(1), need)
    assert torch.isfinite(r["score"]).all()
