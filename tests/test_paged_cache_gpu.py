"""The paged key / value cache on the GPU: appending with rotation and attention over it, against the definitions in 64 bits
(tests/paged_harness.py), at the lengths, layouts and wrong inputs where such kernels go wrong."""
import pytest
import torch

from paged_harness import Case, append_oracle, check_attention, tables

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def run_attention(c, **kw):
    from multimodal_amd import ops
    out = torch.full((c.rows, c.nq, c.hn), 7.0, dtype=c.dtype, device="cuda")
    lse = torch.full((c.rows, c.nq), 7.0, device="cuda")
    kv = c.kv()
    ops.paged_attn_fwd(kv, c.step(**kw), c.q.cuda(), c.scale, out=out, lse=lse)
    torch.cuda.synchronize()
    n = int(c.cu[-1])
    assert bool((out[n:] == 7).all()) and bool((lse[n:] == 7).all()), "rows behind the last sequence were written"
    return out, lse


def run_append(c, cos=None, sin=None, q_out=None):
    from multimodal_amd import ops
    kv = c.kv()
    if q_out is None:
        q_out = torch.full((c.rows, c.nq, c.hn), 7.0, dtype=c.dtype, device="cuda")
    got = ops.paged_kv_append(kv, c.step(), c.k.cuda(), c.v.cuda(), q=c.q.cuda(), cos=None if cos is None else cos.cuda(),
                              sin=None if sin is None else sin.cuda(), q_out=q_out)
    torch.cuda.synchronize()
    assert got is q_out
    return q_out, kv


def check_append(c, q_out, kv, cos=None, sin=None):
    qo, kc, vc, tq, tk = append_oracle(c, cos, sin)
    n = int(c.cu[-1])
    got = q_out[:n].double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(qo[:n]))
    ok = ~torch.isnan(qo[:n])
    assert bool(((got - qo[:n]).abs() <= tq[:n])[ok].all())
    assert bool((q_out[n:] == 7).all()), "rows behind the last sequence were written"
    assert bool(((kv.k.double().cpu() - kc).abs() <= tk).all())
    assert torch.equal(kv.v.double().cpu(), vc)


# ------------------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hn,d,table", [(64, 16, "act"), (64, 64, "fp32"), (128, 32, "fp32"), (128, 128, "act"), (64, 20, "act"),
                                        (128, 2, "fp32"), (64, 0, None)])
def test_append(dtype, hn, d, table):
    c = Case([(1, 1), (0, 9), (5, 17), (33, 40), (1, 64), (0, 0), (2, 2)], nq=6, nkv=3, hn=hn, ps=16, dtype=dtype, pad=3, seed=d)
    cos = sin = None
    if d:
        cos, sin = tables(64, d, torch.float32 if table == "fp32" else dtype)
    check_append(c, *run_append(c, cos, sin), cos, sin)


@pytest.mark.parametrize("ps", [1, 7, 24, 64])
@pytest.mark.parametrize("nseq", [1, 63, 64, 65, 300])
def test_append_page_sizes_and_many_sequences(ps, nseq):
    c = Case([(1 + i % 3 if i % 5 else 0, 3 + (i * 7) % 50) for i in range(nseq)] + [(1, 9)], nq=2, nkv=1, hn=64, ps=ps, dtype=BF16,
             pad=1, seed=nseq)
    cos, sin = tables(64, 16, BF16)
    check_append(c, *run_append(c, cos, sin), cos, sin)


def test_append_in_place_on_the_fused_projection():
    """q, k, v as the slices of [rows, heads, 3, hn], the queries rotated in place."""
    from multimodal_amd import ops
    c = Case([(4, 20), (1, 3)], nq=4, nkv=4, hn=64, ps=16, dtype=BF16)
    cos, sin = tables(32, 16, BF16)
    qkv = torch.stack((c.q, c.k, c.v), dim=2).cuda()
    kv = c.kv()
    q = qkv[:, :, 0]
    assert ops.paged_kv_append(kv, c.step(), qkv[:, :, 1], qkv[:, :, 2], q=q, cos=cos.cuda(), sin=sin.cuda(), q_out=q) is q
    check_append(c, q.clone(), kv, cos, sin)
    assert torch.equal(qkv[:, :, 1].cpu(), c.k) and torch.equal(qkv[:, :, 2].cpu(), c.v)
    # without queries, and with queries of another head count
    kv2 = c.kv()
    assert ops.paged_kv_append(kv2, c.step(), c.k.cuda(), c.v.cuda(), cos=cos.cuda(), sin=sin.cuda()) is None
    assert torch.equal(kv2.k, kv.k) and torch.equal(kv2.v, kv.v)


def test_append_odd_strides_take_the_narrow_path():
    from multimodal_amd import ops
    c = Case([(4, 20), (3, 3)], nq=2, nkv=2, hn=64, ps=16, dtype=F16)
    cos, sin = tables(32, 32, F16)
    wide = torch.zeros(c.rows, 2, 67, dtype=F16, device="cuda")
    k = wide[:, :, 1:65]
    k.copy_(c.k)
    kv = c.kv()
    q = ops.paged_kv_append(kv, c.step(), k, c.v.cuda(), q=c.q.cuda(), cos=cos.cuda(), sin=sin.cuda())
    qf = torch.full_like(q, 7.0)
    qf[:] = q
    check_append(c, qf, kv, cos, sin)


def test_append_rows_without_a_place():
    """Positions below zero, behind the tables and behind the block table, pages the cache does not have: the cache is left
    alone and the query rows are NaN."""
    c = Case([(3, 1), (4, 34), (2, 20), (2, 6)], nq=2, nkv=2, hn=64, ps=8, dtype=BF16, pad=2)
    c.block_table[2, 2] = c.num_pages      # positions 16 .. 23
    c.block_table[3, 0] = -5
    cos, sin = tables(32, 16, BF16)        # positions 32, 33 of sequence 1 have no line
    check_append(c, *run_append(c, cos, sin), cos, sin)
    c = Case([(3, 16), (1, 9)], nq=2, nkv=2, hn=64, ps=8, dtype=BF16)
    c.block_table = c.block_table[:, :1].contiguous()  # positions from 8 on are behind it
    check_append(c, *run_append(c), None, None)


# ---------------------------------------------------------------------------------------------------------- attention
LENGTHS = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 31), (1, 32), (1, 33), (1, 63), (1, 64), (1, 65), (1, 127), (1, 128),
           (1, 129), (1, 130), (0, 40), (1, 257), (0, 0), (1, 700)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hn", [64, 128])
@pytest.mark.parametrize("group,ps", [(1, 16), (4, 64), (16, 24), (3, 1)])
def test_attention_single_tokens(dtype, hn, group, ps):
    c = Case(LENGTHS, nq=2 * group, nkv=2, hn=hn, ps=ps, dtype=dtype, pad=2, seed=group, garbage=float("nan"))
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hn", [64, 128])
@pytest.mark.parametrize("group,ps,seqs", [
    (1, 16, [(1, 1), (2, 2), (7, 9), (16, 16), (3, 33), (0, 5), (16, 50)]),          # at most 16 rows
    (5, 16, [(3, 3), (1, 64), (2, 65), (3, 128)]),
    (1, 16, [(17, 17), (1, 1), (64, 64), (65, 65), (0, 3), (33, 97), (130, 131), (1, 129)]),
    (4, 64, [(32, 32), (33, 70), (40, 300), (1, 2)]),
    (3, 24, [(50, 120), (43, 43)]),
    (2, 128, [(129, 130)]),
])
def test_attention_chunks(dtype, hn, group, ps, seqs):
    c = Case(seqs, nq=2 * group, nkv=2, hn=hn, ps=ps, dtype=dtype, pad=1, seed=ps, garbage=float("inf"))
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("hn", [64, 128])
@pytest.mark.parametrize("seqs", [[(1, 5000), (1, 3), (1, 1025), (0, 0)], [(9, 4001), (2, 2)], [(40, 3000), (1, 600), (20, 20)]])
def test_attention_long_axis_is_split(hn, seqs):
    from multimodal_amd._lib import get_lib
    c = Case(seqs, nq=4, nkv=2, hn=hn, ps=32, dtype=BF16, pad=1, garbage=float("nan"))
    step, kv = c.step(), c.kv()
    assert get_lib().mm_paged_attn_workspace_bytes(kv._ref, step._ref, c.nq, c.rows) > 0
    check_attention(c, *run_attention(c))
    # bounds larger than the lengths: other splits, the same rows
    check_attention(c, *run_attention(c, max_kv=c.max_kv + 70000, max_new=c.max_new))


@pytest.mark.parametrize("hn", [64, 128])
@pytest.mark.parametrize("n,l", [(5, 2), (16, 0), (40, 10), (70, 1)])
def test_attention_rows_that_see_no_key(hn, n, l):
    c = Case([(n, l), (2, 9)], nq=2, nkv=2, hn=hn, ps=16, dtype=BF16, garbage=float("nan"))
    check_attention(c, *run_attention(c))
    check_attention(c, *run_attention(c, max_kv=5000))


@pytest.mark.parametrize("hn", [64, 128])
@pytest.mark.parametrize("n,l", [(1, 90), (6, 90), (16, 33), (33, 90), (90, 90), (150, 700)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_attention_nonfinite_keys_and_values_reach_only_rows_that_see_them(hn, n, l, value):
    """A value that is not finite shows in its dim of the rows that see it and nowhere else; a NaN key makes the rows that see
    it NaN."""
    c = Case([(n, l), (3, 20)], nq=2, nkv=1, hn=hn, ps=16, dtype=BF16)
    for p, d in ((l - 1, 3), (max(0, l - n // 2 - 1), hn - 1), (max(0, l - n), 17)):
        c.v_cache[c.block_table[0, p // 16], 0, p % 16, d] = value
    check_attention(c, *run_attention(c))
    c.k_cache[c.block_table[0, (l - 1) // 16], 0, (l - 1) % 16, 5] = float("nan")
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("n", [1, 40])
def test_attention_pages_the_cache_does_not_have(n):
    c = Case([(n, 130), (n, 90), (n, 64)], nq=2, nkv=2, hn=64, ps=16, dtype=BF16)
    c.block_table[0, 6] = c.num_pages
    c.block_table[1, 5] = -1
    c.block_table[2, 0] = 2 ** 31 - 1
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("max_new,max_kv", [(2, 4000), (5, 60), (1, 10)])
def test_attention_broken_bounds_give_nan(max_new, max_kv):
    """A sequence beyond the step's bounds is NaN as a whole, the others are right."""
    c = Case([(1, 50), (5, 55), (2, 3000), (1, 4)], nq=2, nkv=2, hn=64, ps=16, dtype=BF16, pad=1)
    out, lse = run_attention(c, max_new=max_new, max_kv=max_kv)
    good = []
    for i, (n, l) in enumerate(c.seqs):
        a, b = int(c.cu[i]), int(c.cu[i + 1])
        if n > max_new or l > max_kv:
            assert bool(torch.isnan(out[a:b]).all()) and bool(torch.isnan(lse[a:b]).all())
        else:
            good.append(i)
            ref_out, ref_lse = run_attention(c)
            assert torch.allclose(out[a:b].float(), ref_out[a:b].float(), rtol=2.0 ** -6, atol=2.0 ** -6)
    assert good


def test_layouts_and_views_of_the_cache():
    """Slot-major pages, keys and values in one tensor, a block table that is a view: the same bits as the packed layout."""
    from multimodal_amd import ops
    from multimodal_amd.kv_cache import PagedKV, PagedStep
    c = Case([(1, 70), (20, 90), (0, 10), (2, 2)], nq=4, nkv=2, hn=64, ps=16, dtype=BF16)
    ref = run_attention(c)
    both = torch.zeros(c.num_pages, 2, c.ps, c.nkv, c.hn + 8, dtype=BF16, device="cuda")
    k = both[:, 0, :, :, :c.hn].transpose(1, 2)
    v = both[:, 1, :, :, 8:].transpose(1, 2)
    k.copy_(c.k_cache)
    v.copy_(c.v_cache)
    bt = torch.full((4, 40), -9, dtype=torch.int32, device="cuda")
    bt[:, 3:3 + c.block_table.size(1)] = c.block_table.cuda()
    step = PagedStep(bt[:, 3:3 + c.block_table.size(1)], c.cu.cuda(), c.lens.cuda(), c.max_new, c.max_kv)
    q = torch.zeros(c.rows, 4, 3, c.hn, dtype=BF16, device="cuda")
    q[:, :, 1] = c.q.cuda()
    out, lse = ops.paged_attn_fwd(PagedKV(k, v), step, q[:, :, 1], c.scale)
    assert torch.equal(out, ref[0]) and torch.equal(lse, ref[1])
    # odd alignment of the queries: copied by the wrapper
    flat = torch.zeros(c.rows * 4 * c.hn + 1, dtype=BF16, device="cuda")
    q1 = flat[1:].view(c.rows, 4, c.hn)
    q1.copy_(c.q)
    out, lse = ops.paged_attn_fwd(PagedKV(k, v), step, q1, c.scale)
    assert torch.equal(out, ref[0]) and torch.equal(lse, ref[1])


def test_offsets_beyond_32_bits():
    """Pages whose element offsets pass 2^32."""
    from multimodal_amd import ops
    from multimodal_amd.kv_cache import PagedKV
    c = Case([(1, 100), (20, 50)], nq=16, nkv=16, hn=128, ps=64, dtype=BF16)
    pages = (1 << 32) // (16 * 64 * 128) + 8
    base = pages - c.num_pages
    big_k = torch.empty(pages, 16, 64, 128, dtype=BF16, device="cuda")
    big_v = torch.empty(pages, 16, 64, 128, dtype=BF16, device="cuda")
    big_k[base:] = c.k_cache.cuda()
    big_v[base:] = c.v_cache.cuda()
    kv = PagedKV(big_k, big_v)
    table = c.block_table.clone()
    c.block_table = torch.where(table >= 0, table + base, table)
    step = c.step()
    c.block_table = table
    cos, sin = tables(128, 128, BF16)
    q_out = ops.paged_kv_append(kv, step, c.k.cuda(), c.v.cuda(), q=c.q.cuda(), cos=cos.cuda(), sin=sin.cuda())
    small = c.kv()
    assert torch.equal(q_out, ops.paged_kv_append(small, c.step(), c.k.cuda(), c.v.cuda(), q=c.q.cuda(), cos=cos.cuda(), sin=sin.cuda()))
    assert torch.equal(big_k[base:], small.k) and torch.equal(big_v[base:], small.v)
    a, b = ops.paged_attn_fwd(kv, step, q_out, c.scale), ops.paged_attn_fwd(small, c.step(), q_out, c.scale)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    del big_k, big_v, kv
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------- streams, graphs, repetition
@pytest.mark.parametrize("seqs", [[(1, 3000), (1, 70)], [(40, 2000), (3, 3)]])
def test_same_bits_twice_on_another_stream_and_in_a_replayed_graph(seqs):
    from multimodal_amd import ops
    c = Case(seqs, nq=4, nkv=2, hn=64, ps=16, dtype=BF16, pad=2)
    kv, step, q = c.kv(), c.step(), c.q.cuda()
    k, v = c.k.cuda(), c.v.cuda()
    cos, sin = (t.cuda() for t in tables(4000, 16, BF16))

    def once():
        qo = ops.paged_kv_append(kv, step, k, v, q=q, cos=cos, sin=sin)
        return ops.paged_attn_fwd(kv, step, qo, c.scale)

    n = int(c.cu[-1])
    ref = [t[:n].clone() for t in once()]
    again = once()
    assert all(torch.equal(x[:n], y) for x, y in zip(again, ref))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x[:n], y) for x, y in zip(other, ref))
    # two captured graphs, replayed in turn with eager calls and new inputs between the replays
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = once()
        graphs.append((g, res))
    for rep in range(4):
        with torch.no_grad():
            q.copy_(c.q.cuda() * (1.0 + rep))
            k.copy_(c.k.cuda() * (0.5 + rep))
            if rep == 2:  # the step's arrays are read at run time: shorter sequences
                step.kv_lens.copy_((c.lens - 1).cuda())
        eager = [t[:n].clone() for t in once()]
        for g, res in graphs:
            for t in res:
                t.fill_(3.0)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x[:n], y) for x, y in zip(res, eager)), f"replay {rep}"


# ------------------------------------------------------------------------- values that are not finite where every row sees them
@pytest.mark.parametrize("hn,dtype", [(64, F16), (128, BF16), (128, F16)])
@pytest.mark.parametrize("n,l", [(1, 90), (6, 300), (1, 5000), (40, 300), (150, 700), (40, 3000)])
@pytest.mark.parametrize("spread", [1.0, 60.0])
def test_attention_nonfinite_values_that_every_row_sees(hn, dtype, n, l, spread):
    """p > 0 times an infinity is that infinity, also where p rounds to 0 (in 16 bits or, at the wide spread of scores, in 32) and
    whichever split or wave it meets; infinities of both signs or a NaN in one dim make it NaN."""
    c = Case([(n, l), (3, 200), (1, 33)], nq=2, nkv=1, hn=hn, ps=16, dtype=dtype)
    c.q = (c.q.float() * spread).to(dtype)
    inf = float("inf")
    for p, d, x in ((2, 3, inf), (37, 3, inf), (41, 9, -inf), (70, 20, inf), (11, 20, -inf), (l - n, hn - 1, float("nan"))):
        c.v_cache[c.block_table[0, p // 16], 0, p % 16, d] = x
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("n", [1, 40])
def test_attention_lengths_below_zero(n):
    """A length below the new rows, down to the smallest number: the rows see nothing."""
    c = Case([(n, -3), (n, 100), (n, -2 ** 31)], nq=2, nkv=2, hn=64, ps=16, dtype=BF16, pad=1, garbage=float("nan"))
    check_attention(c, *run_attention(c))
    check_attention(c, *run_attention(c, max_kv=9000))


def test_nothing_to_do():
    """No rows, no sequences, sequences without rows: nothing is written and nothing fails."""
    from multimodal_amd import ops
    from multimodal_amd.kv_cache import PagedStep
    c = Case([(0, 5), (0, 40)], nq=4, nkv=2, hn=64, ps=16, dtype=BF16)
    for step in (c.step(), PagedStep(torch.empty(0, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
                                     torch.empty(0, dtype=torch.int32, device="cuda"))):
        kv = c.kv()
        kv_rows = torch.empty(0, 2, 64, dtype=BF16, device="cuda")
        q = torch.empty(0, 4, 64, dtype=BF16, device="cuda")
        assert ops.paged_kv_append(kv, step, kv_rows, kv_rows.clone(), q=q).shape == (0, 4, 64)
        assert ops.paged_kv_append(kv, step, kv_rows, kv_rows.clone()) is None
        out, lse = ops.paged_attn_fwd(kv, step, q, c.scale)
        assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
        torch.cuda.synchronize()
        assert torch.equal(kv.k.cpu(), c.k_cache) and torch.equal(kv.v.cpu(), c.v_cache)


def test_outputs_that_overlap_themselves_are_refused():
    from multimodal_amd import ops
    c = Case([(2, 9)], nq=2, nkv=2, hn=64, ps=16, dtype=BF16)
    one = torch.zeros(1, 2, 64, dtype=BF16, device="cuda").expand(2, 2, 64)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.paged_attn_fwd(c.kv(), c.step(), c.q.cuda(), c.scale, out=one)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.paged_attn_fwd(c.kv(), c.step(), c.q.cuda(), c.scale, lse=torch.zeros(1, 2, device="cuda").expand(2, 2))
    with pytest.raises(RuntimeError, match="overlap"):
        ops.paged_kv_append(c.kv(), c.step(), c.k.cuda(), c.v.cuda(), q=c.q.cuda(), q_out=one)


def test_cache_steps_that_make_no_sense_are_refused():
    from multimodal_amd.kv_cache import PagedKVCache, PagedStep
    cache = PagedKVCache(1, 2, 64, num_pages=8, page_size=4)
    a, b = cache.add(8), cache.add(3)
    with pytest.raises(RuntimeError, match="twice"):
        cache.step([a, b, a], [1, 1, 1], [3, 2, 4])
    with pytest.raises(RuntimeError, match="numbers"):
        cache.step([a, b], [1], [3, 2])
    with pytest.raises(RuntimeError, match="no sequence"):
        cache.step([a, 99], [1, 1], [3, 2])
    for bad in (lambda: cache.release(99), lambda: cache.reserve(99, 4), lambda: cache.block_table([99])):
        with pytest.raises(RuntimeError, match="no sequence"):
            bad()
    cache.release(b)
    with pytest.raises(RuntimeError, match="no sequence"):
        cache.release(b)
    assert cache.free_pages == 6
    s = cache.step([a], [1], [3])
    with pytest.raises(RuntimeError, match="max_kv"):
        PagedStep(s.block_table, s.cu_new, s.kv_lens, max_new=1, max_kv=2 ** 32 + 3)


@pytest.mark.parametrize("hn,dtype", [(64, BF16), (128, F16)])
@pytest.mark.parametrize("group,ps", [(1, 16), (16, 24), (3, 1)])
@pytest.mark.parametrize("max_kv", [10000, 1000000])
def test_attention_single_tokens_under_larger_bounds(hn, dtype, group, ps, max_kv):
    """Bounds far above the lengths: larger workgroups and splits that hold no key, the same rows."""
    c = Case(LENGTHS, nq=2 * group, nkv=2, hn=hn, ps=ps, dtype=dtype, pad=2, seed=group, garbage=float("inf"))
    check_attention(c, *run_attention(c, max_kv=max_kv))


def test_two_streams_at_once():
    """Calls in flight together, each with a workspace of its own, over one cache: the bits of a call alone."""
    from multimodal_amd import ops
    cases = [Case([(1, 3000), (1, 70), (2, 900)], nq=4, nkv=2, hn=64, ps=16, dtype=BF16, seed=1),
             Case([(40, 2000), (1, 1500)], nq=4, nkv=2, hn=64, ps=16, dtype=BF16, seed=2)]
    ready = [(c.kv(), c.step(), c.q.cuda(), c.scale) for c in cases]
    ref = [ops.paged_attn_fwd(*r) for r in ready]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, r in enumerate(ready):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.paged_attn_fwd(*r))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, ref[i][0]) and torch.equal(l, ref[i][1]) for o, l in got[i])


@pytest.mark.parametrize("nq,nkv,hn,d", [(4, 1, 64, 16), (26, 4, 128, 128), (4, 2, 64, 20), (16, 16, 64, 16)])
def test_append_many_rows_equals_few(nq, nkv, hn, d):
    """Thousands of rows in one call - sequences without rows between them, padding, rows without a place - against the same rows a
    few hundred at a time: the same bits."""
    from multimodal_amd import ops
    from multimodal_amd.kv_cache import PagedStep
    g = torch.Generator().manual_seed(nq)
    n = torch.randint(0, 90, (240,), generator=g)
    n[20:32] = 0   # a run of sequences without rows
    n[100:103] = 0
    seqs = [(int(x), int(x) + int(p)) for x, p in zip(n, torch.randint(0, 40, (240,), generator=g))]
    c = Case(seqs, nq=nq, nkv=nkv, hn=hn, ps=16, dtype=BF16, pad=5, seed=d)
    assert c.rows > 8 * 1024 + 64
    c.block_table[50, 0] = c.num_pages
    c.block_table[51, 1:] = -1
    cos, sin = (t.cuda() for t in tables(110, d, BF16))  # some positions lie behind them
    k, v, q = c.k.cuda(), c.v.cuda(), c.q.cuda()
    many, few = c.kv(), c.kv()
    out = torch.full((c.rows, nq, hn), 7.0, dtype=BF16, device="cuda")
    ref = out.clone()
    ops.paged_kv_append(many, c.step(), k, v, q=q, cos=cos, sin=sin, q_out=out)
    for a in range(0, 240, 8):
        r0, r1 = int(c.cu[a]), int(c.cu[a + 8])
        step = PagedStep(c.block_table[a:a + 8].cuda(), (c.cu[a:a + 9] - r0).cuda(), c.lens[a:a + 8].cuda(), c.max_new, c.max_kv)
        ops.paged_kv_append(few, step, k[r0:r1], v[r0:r1], q=q[r0:r1], cos=cos, sin=sin, q_out=ref[r0:r1])
    assert torch.equal(torch.isnan(out), torch.isnan(ref)) and torch.equal(out.nan_to_num(), ref.nan_to_num())
    assert bool(torch.isnan(out).any()) and bool((out[int(c.cu[-1]):] == 7).all())
    assert torch.equal(many.k, few.k) and torch.equal(many.v, few.v)


def test_outputs_beside_their_inputs():
    """q_out in a slot of its own in the fused projection, out in the queries' place: the bits of outputs apart; outputs that meet their
    inputs otherwise are refused."""
    from multimodal_amd import ops
    for seqs in ([(4, 20), (1, 3)], [(1, 3000), (3, 500)], [(40, 60), (70, 3000)]):
        c = Case(seqs, nq=4, nkv=4, hn=64, ps=16, dtype=BF16)
        cos, sin = (t.cuda() for t in tables(3000, 16, BF16))
        kv, step = c.kv(), c.step()
        ref_q = ops.paged_kv_append(kv, step, c.k.cuda(), c.v.cuda(), q=c.q.cuda(), cos=cos, sin=sin)
        ref = ops.paged_attn_fwd(kv, step, ref_q, c.scale)
        four = torch.stack((c.q, c.k, c.v, torch.zeros_like(c.q)), dim=2).cuda()
        q, k, v, out = four.unbind(2)
        assert torch.equal(ops.paged_kv_append(kv, step, k, v, q=q, cos=cos, sin=sin, q_out=out), ref_q)
        assert torch.equal(q.cpu(), c.q) and torch.equal(k.cpu(), c.k) and torch.equal(v.cpu(), c.v)
        got = ops.paged_attn_fwd(kv, step, out, c.scale, out=q)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        got = ops.paged_attn_fwd(kv, step, out, c.scale, out=out)
        assert torch.equal(out, ref[0]) and torch.equal(got[1], ref[1])
        wide = torch.zeros(c.rows + 1, 4, 64, dtype=BF16, device="cuda")
        with pytest.raises(RuntimeError, match="in part"):
            ops.paged_attn_fwd(kv, step, wide[:-1], c.scale, out=wide[1:])
        with pytest.raises(RuntimeError, match="in part"):
            ops.paged_kv_append(kv, step, k, v, q=wide[:-1], q_out=wide[1:])
        with pytest.raises(RuntimeError, match="k or v"):
            ops.paged_kv_append(kv, step, k, v, q=c.q.cuda(), q_out=v)
        with pytest.raises(RuntimeError, match="lse overlaps"):
            ops.paged_attn_fwd(kv, step, wide[:-1], c.scale, lse=wide.view(-1).view(torch.float32)[:c.rows * 4].view(c.rows, 4))


def test_operands_that_want_a_gradient_are_refused():
    """There is no backward: a gradient would stop here without a word."""
    from multimodal_amd import ops
    c = Case([(2, 9)], nq=2, nkv=2, hn=64, ps=16, dtype=BF16)
    kv, step = c.kv(), c.step()
    k, v, q = c.k.cuda(), c.v.cuda(), c.q.cuda()
    for which in range(3):
        t = [k, v, q]
        t[which] = t[which].clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="no backward"):
            ops.paged_kv_append(kv, step, t[0], t[1], q=t[2])
        with torch.no_grad():
            ops.paged_kv_append(kv, step, t[0], t[1], q=t[2])
    with pytest.raises(RuntimeError, match="no backward"):
        ops.paged_attn_fwd(kv, step, q.clone().requires_grad_(True), c.scale)
    with torch.no_grad():
        ops.paged_attn_fwd(kv, step, q.clone().requires_grad_(True), c.scale)


# --------------------------------------------------------------------------- calls that the documentation allows, less usual ones
@pytest.mark.parametrize("hn,dtype", [(64, BF16), (128, F16)])
@pytest.mark.parametrize("group,nkv", [(17, 1), (32, 2), (71, 1)])
def test_attention_single_tokens_of_many_heads_a_key(hn, dtype, group, nkv):
    """More than 16 query heads on a key head: single tokens in the form of chunks, in one piece and split."""
    c = Case([(1, 1), (1, 40), (0, 7), (1, 200), (2, 65)], nq=group * nkv, nkv=nkv, hn=hn, ps=16, dtype=dtype, pad=1, garbage=float("nan"))
    check_attention(c, *run_attention(c))
    check_attention(c, *run_attention(c, max_kv=6000))


@pytest.mark.parametrize("hn", [64, 128])
@pytest.mark.parametrize("ps", [1, 7, 300])
def test_attention_chunks_over_pages_of_any_size(hn, ps):
    c = Case([(40, 130), (17, 17), (1, 90), (70, 71), (20, 300)], nq=4, nkv=2, hn=hn, ps=ps, dtype=BF16, pad=1, garbage=float("inf"))
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("seqs,max_kv", [([(1, 70), (2, 9), (1, 400)], 0), ([(1, 3000), (1, 70)], 0), ([(40, 300), (2, 9)], 0),
                                         ([(40, 1500), (1, 700)], 9000)])
def test_attention_outputs_in_wider_tensors(seqs, max_kv):
    """Outputs as slices of wider tensors, whose other elements stay; rows ahead of the first sequence stay too."""
    from multimodal_amd import ops
    from multimodal_amd.kv_cache import PagedStep
    c = Case(seqs, nq=4, nkv=2, hn=64, ps=16, dtype=BF16, pad=2, garbage=float("nan"))
    ref = run_attention(c, **(dict(max_kv=max_kv) if max_kv else {}))
    n, ahead = int(c.cu[-1]), 3
    step = PagedStep(c.block_table.cuda(), (c.cu + ahead).cuda(), c.lens.cuda(), c.max_new, max_kv or c.max_kv)
    q = torch.cat((torch.full((ahead, 4, 64), float("nan"), dtype=BF16), c.q)).cuda()
    wide = torch.full((ahead + c.rows, 4, 3, 72), 7.0, dtype=BF16, device="cuda")
    lse = torch.full((ahead + c.rows, 9), 7.0, device="cuda")
    ops.paged_attn_fwd(c.kv(), step, q, c.scale, out=wide[:, :, 1, 8:], lse=lse[:, 2:6])
    assert torch.equal(wide[ahead:ahead + n, :, 1, 8:], ref[0][:n]) and torch.equal(lse[ahead:ahead + n, 2:6], ref[1][:n])
    wide[ahead:ahead + n, :, 1, 8:] = 7.0
    lse[ahead:ahead + n, 2:6] = 7.0
    assert bool((wide == 7).all()) and bool((lse == 7).all())
    # the append leaves them alone as well
    kv, kv2 = c.kv(), c.kv()
    cos, sin = (t.cuda() for t in tables(3000, 16, BF16))
    k, v = (torch.cat((t[:ahead], t)).cuda() for t in (c.k, c.v))
    qo = torch.full((ahead + c.rows, 4, 64), 7.0, dtype=BF16, device="cuda")
    ops.paged_kv_append(kv, step, k, v, q=q, cos=cos, sin=sin, q_out=qo)
    want = ops.paged_kv_append(kv2, c.step(), c.k.cuda(), c.v.cuda(), q=c.q.cuda(), cos=cos, sin=sin)
    assert torch.equal(kv.k.nan_to_num(), kv2.k.nan_to_num()) and torch.equal(kv.v.nan_to_num(), kv2.v.nan_to_num())
    assert torch.equal(qo[ahead:ahead + n], want[:n]) and bool((qo[:ahead] == 7).all()) and bool((qo[ahead + n:] == 7).all())


def test_thousands_of_sequences():
    """More sequences than two steps of the search for a row's sequence cover, some without rows; and many that are split and joined."""
    c = Case([(1 + (i % 7 == 3) if i % 5 else 0, 3 + (i * 7) % 50) for i in range(4500)], nq=1, nkv=1, hn=64, ps=16, dtype=BF16, pad=1, seed=3)
    cos, sin = tables(64, 16, BF16)
    check_append(c, *run_append(c, cos, sin), cos, sin)
    check_attention(c, *run_attention(c))
    c = Case([(17 + i % 3 if i % 4 else 1, 20 + (i * 37) % 1100) for i in range(100)], nq=1, nkv=1, hn=64, ps=16, dtype=BF16, pad=1, seed=4)
    from multimodal_amd._lib import get_lib
    step, kv = c.step(), c.kv()
    assert get_lib().mm_paged_attn_workspace_bytes(kv._ref, step._ref, c.nq, c.rows) > 0
    check_attention(c, *run_attention(c))


def test_a_replayed_step_follows_its_arrays():
    """Pages, rows and lengths of a captured step are rewritten between the replays, a broken step among them."""
    from multimodal_amd import ops
    steps = [[(1, 300), (3, 700), (0, 20)], [(2, 40), (1, 1500), (1, 1)], [(0, 9), (4, 1499), (0, 0)], [(3, 2000), (1, 5), (0, 3)], [(1, 1), (1, 2), (2, 3)]]
    cases = [Case(s, nq=4, nkv=2, hn=64, ps=16, dtype=BF16, seed=i) for i, s in enumerate(steps)]
    pages, width = max(c.num_pages for c in cases), 94  # 1504 positions: the fourth step's 2000 are behind the table
    table = torch.zeros(3, width, dtype=torch.int32, device="cuda")
    cu, lens = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    from multimodal_amd.kv_cache import PagedKV, PagedStep
    kv = PagedKV(torch.zeros(pages, 2, 16, 64, dtype=BF16, device="cuda"), torch.zeros(pages, 2, 16, 64, dtype=BF16, device="cuda"))
    step = PagedStep(table, cu, lens, max_new=4, max_kv=1504)
    q = torch.zeros(4, 4, 64, dtype=BF16, device="cuda")
    out, lse = torch.zeros(4, 4, 64, dtype=BF16, device="cuda"), torch.zeros(4, 4, device="cuda")
    ops.paged_attn_fwd(kv, step, q, 0.125, out=out, lse=lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attn_fwd(kv, step, q, 0.125, out=out, lse=lse)
    for c in cases + cases[::-1]:
        bt = torch.full((3, width), -1, dtype=torch.int32)
        w = min(width, c.block_table.size(1))
        bt[:, :w] = c.block_table[:, :w]
        table.copy_(bt)
        cu.copy_(c.cu)
        lens.copy_(c.lens)
        kv.k[:c.num_pages].copy_(c.k_cache)
        kv.v[:c.num_pages].copy_(c.v_cache)
        n = int(c.cu[-1])
        q[:n].copy_(c.q[:n])
        out.fill_(7.0)
        lse.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert bool((out[n:] == 7).all()) and bool((lse[n:] == 7).all())
        if int(c.lens.max()) > 1504:
            assert bool(torch.isnan(out[:3]).all()) and bool(torch.isnan(lse[:3]).all()) and not bool(torch.isnan(out[3]).any())
        else:
            check_attention(c, out, lse)
