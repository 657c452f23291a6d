"""Turned rows over what the same launch reads: refused, and what lies beside it is not."""

import pytest

import serving

pytestmark = pytest.mark.gpu


def test_outputs_over_what_is_read(gpu):
    import torch
    import fusor_kernels as fk
    for rows in (1, 2, 40):
        step = serving.Step([rows], [rows])
        rotary, batch, cache = fk.Rotary(16), step.batch(fk, gpu), fk.PagedCache(step.pages, 2, 16, device=gpu)
        flat = torch.randn(rows, 200, device=gpu)  # [rows, 12.5 heads]
        heads = lambda first, count: flat[:, 16 * first:16 * (first + count)].unflatten(1, (count, 16))
        keys, values, queries = heads(0, 2), heads(2, 2), heads(4, 2)
        before = flat.clone()
        for out in (keys, values, heads(1, 2), heads(3, 2)):
            with pytest.raises(fk.ShapeError, match="lie over"):  # (the last lies over the queries too)
                cache.write(batch, keys, values, rotary=rotary, queries=queries, out=out)
        with pytest.raises(fk.ShapeError, match="over the keys or values"):
            cache.write(batch, keys, values, rotary=rotary, queries=keys, out=keys)
        for out in (heads(3, 2), heads(5, 2)):
            with pytest.raises(fk.ShapeError, match="a part of the rows"):
                rotary.rotate(batch, queries, out=out)
        if rows > 2:  # a row down
            with pytest.raises(fk.ShapeError, match="a part of the rows"):
                short = serving.Step([rows - 1], [rows - 1])
                rotary.rotate(short.batch(fk, gpu), queries[1:], out=queries[:-1])  # (the same rows, one up)
        torch.cuda.synchronize()
        assert torch.equal(flat, before)
        # beside the keys, the values and the queries, in the same rows; and in place
        out = heads(6, 2)
        cache.write(batch, keys, values, rotary=rotary, queries=queries, out=out)
        want = rotary.rotate(batch, before[:, 64:96].unflatten(1, (2, 16)).contiguous())
        assert torch.equal(out, want)
        rotary.rotate(batch, queries, out=heads(8, 2))
        assert torch.equal(heads(8, 2), want)
        cache.write(batch, keys, values, rotary=rotary, queries=queries, out=queries)
        assert torch.equal(queries, want) and torch.equal(flat[:, :64], before[:, :64])
        got = [torch.zeros(rows, 2, 16, device=gpu) for _ in range(2)]
        cache.read(batch, *got)
        assert torch.equal(got[0].cpu(), serving.quantized(rotary.rotate(batch, keys.contiguous()).cpu()).float())
        # outputs behind all of the rows, with another stride
        apart = torch.zeros(rows, 2, 16, device=gpu)
        assert cache.write(batch, keys, values, rotary=rotary, queries=heads(6, 2), out=apart) is apart
