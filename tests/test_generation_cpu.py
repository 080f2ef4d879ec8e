"""Refusals of the generation entry points, before any device work: safe without a GPU."""
import ctypes

import pytest
import torch

from multimodal_amd import _lib, ops
from multimodal_amd._lib import MmPagedKV, MmPagedStep

KV = dict(k=4096, v=8192, page=4 * 16 * 64, head=16 * 64, slot=64, num_pages=10, page_size=16, heads=4, hn=64, dtype=0)
STEP = dict(block_table=4096, cu_new=4096, kv_lens=4096, table_stride=8, seqs=2, max_pages=8, max_new=1, max_kv=100)


def refs(kv=(), step=()):
    a, b = MmPagedKV(**{**KV, **dict(kv)}), MmPagedStep(**{**STEP, **dict(step)})
    return a, b, ctypes.addressof(a), ctypes.addressof(b)


def append(kv=(), step=(), k=4096, v=4096, q=4096, q_out=4096, nq=4, rows=2, cos=4096, sin=4096, d=16, positions=100):
    a, b, pa, pb = refs(kv, step)
    lib = _lib.get_lib()
    return lib.mm_paged_kv_append(pa, pb, k, 256, 64, v, 256, 64, q, 256, 64, q_out, 256, 64, nq, rows, cos, sin, d, positions, 1, None), \
        lib.mm_last_error().decode()


def attend(kv=(), step=(), out=4096, lse=4096, q=4096, q_row=256, nq=4, rows=2, scale=0.125, ws=0, ws_bytes=0):
    a, b, pa, pb = refs(kv, step)
    lib = _lib.get_lib()
    return lib.mm_paged_attn_fwd(pa, pb, out, 256, 64, lse, nq, q, q_row, 64, nq, rows, scale, ws, ws_bytes, None), \
        lib.mm_last_error().decode()


BAD_CACHE = [(dict(k=0), "null"), (dict(hn=96), "head size"), (dict(num_pages=0), "out of range"), (dict(page_size=0), "out of range"),
             (dict(heads=-1), "out of range"), (dict(k=4100), "16-byte"), (dict(page=1 << 31), "stride"), (dict(head=12), "stride"),
             (dict(slot=0), "stride"), (dict(slot=-64), "stride"), (dict(page_size=1 << 20, slot=4096), "slots span")]
BAD_STEP = [(dict(block_table=0), "null"), (dict(cu_new=0), "null"), (dict(kv_lens=0), "null"), (dict(seqs=-1), "out of range"),
            (dict(max_pages=0), "out of range"), (dict(max_pages=1 << 27, table_stride=1 << 27), "2^30"), (dict(max_new=-1), "out of range"),
            (dict(max_kv=-1), "out of range"), (dict(table_stride=7), "out of range")]


@pytest.mark.parametrize("call", [append, attend])
def test_bad_caches_and_steps(call):
    for bad, text in BAD_CACHE:
        rc, msg = call(kv=bad)
        assert rc == -1 and text in msg, (bad, rc, msg)
    for bad, text in BAD_STEP:
        rc, msg = call(step=bad)
        assert rc == -1 and text in msg, (bad, rc, msg)


def test_bad_append_arguments():
    for bad, text in [(dict(k=0), "null"), (dict(v=0), "null"), (dict(q_out=0), "q_out"), (dict(nq=0), "head count"), (dict(d=15), "rotary"),
                      (dict(d=66), "rotary"), (dict(d=-2), "rotary"), (dict(cos=0), "tables"), (dict(positions=0), "tables"), (dict(rows=-1), "out of range")]:
        rc, msg = append(**bad)
        assert rc == -1 and text in msg, (bad, rc, msg)
    rc, msg = append(kv=dict(dtype=7))
    assert rc == -2 and "dtype" in msg
    assert append(rows=0)[0] == 0 and append(step=dict(seqs=0))[0] == 0  # nothing to do is no error


def test_bad_attention_arguments():
    for bad, text in [(dict(out=0), "null"), (dict(lse=0), "null"), (dict(q=0), "null"), (dict(nq=6), "multiple"), (dict(nq=0), "multiple"),
                      (dict(q=4104), "aligned"), (dict(q_row=252), "aligned"), (dict(scale=0.0), "softmax_scale"), (dict(scale=float("nan")), "softmax_scale"),
                      (dict(step=dict(max_kv=1 << 30)), "2^30"), (dict(step=dict(max_new=1 << 30)), "grid")]:
        rc, msg = attend(**bad)
        assert rc == -1 and text in msg, (bad, rc, msg)
    assert attend(kv=dict(dtype=7))[0] == -2
    assert attend(rows=0)[0] == 0 and attend(step=dict(max_new=0))[0] == 0


def test_workspace_is_asked_for_and_checked():
    a, b, pa, pb = refs(step=dict(max_kv=5000, max_pages=512, table_stride=512))
    lib = _lib.get_lib()
    need = lib.mm_paged_attn_workspace_bytes(pa, pb, 4, 2)
    assert need > 0 and need % (2 * 4 * 66 * 4) == 0
    for ws, n in ((0, need), (4096, need - 1), (4100, need)):
        rc, msg = attend(step=dict(max_kv=5000, max_pages=512, table_stride=512), ws=ws, ws_bytes=n)
        assert rc == -1 and "workspace" in msg
    a, b, pa, pb = refs()
    assert lib.mm_paged_attn_workspace_bytes(pa, pb, 4, 2) == 0          # short: in one piece
    assert lib.mm_paged_attn_workspace_bytes(pa, pb, 5, 2) == 0          # not a call attention would take


def test_bad_sampling_arguments():
    lib = _lib.get_lib()

    def call(tokens=4096, logits=4096, u=4096, rows=2, vocab=100, dtype=0):
        return lib.mm_sample_tokens(tokens, logits, 128, u, rows, vocab, 1.0, None, 0, None, 0.0, None, 0.0, None, dtype, None), \
            lib.mm_last_error().decode()
    for bad, text in [(dict(tokens=0), "null"), (dict(logits=0), "null"), (dict(u=0), "null"), (dict(rows=-1), "out of range"),
                      (dict(vocab=0), "out of range"), (dict(vocab=1 << 30), "out of range"), (dict(logits=4097), "aligned")]:
        rc, msg = call(**bad)
        assert rc == -1 and text in msg, (bad, rc, msg)
    assert call(dtype=3)[0] == -2 and call(rows=0)[0] == 0


def test_wrappers_refuse_cpu_tensors():
    from multimodal_amd.kv_cache import PagedKV, PagedStep
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        PagedKV(k, k.clone())
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="one GPU"):
        PagedStep(torch.zeros(1, 4, dtype=torch.int32), i, i[:1])
    with pytest.raises(RuntimeError, match="GPU"):
        ops.sample_tokens(torch.zeros(2, 100, dtype=torch.bfloat16), torch.zeros(2))


@pytest.mark.parametrize("d", [1, 2, 3, 7, 8, 16, 24, 48, 63, 64, 100, 128, 1000, 65536, (1 << 20) + 1])
def test_division_by_multiplication(d):
    """The kernels' n / page_size: (mulhi(m, n) + n) >> l with l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1, exact below 2^31."""
    l = (d - 1).bit_length()
    m = (((1 << l) - d) << 32) // d + 1
    assert m < 1 << 32
    ns = {0, 1, d - 1, d, d + 1, (1 << 31) - 1, (1 << 30) - 1}
    ns |= {k * d + e for k in (1, 2, 1000, ((1 << 31) - 1) // d) for e in (-1, 0, 1)}
    for n in ns:
        if 0 <= n < 1 << 31:
            q = ((m * n) >> 32) + n
            assert q < 1 << 32 and q >> l == n // d, (n, d)


def test_launches_beyond_the_grid_are_refused():
    """A grid dimension times the workgroup's threads stays below 2^32."""
    lib = _lib.get_lib()
    rc, msg = append(rows=(1 << 31) - 1)
    assert rc == -1 and "grid" in msg
    rc, msg = attend(step=dict(seqs=1 << 21))
    assert rc == -1 and "grid" in msg
    big = dict(max_kv=5000, max_new=100, max_pages=512, table_stride=512, seqs=1)  # the long axis is split, and its rows joined
    a, b, pa, pb = refs(step=big)
    need = lib.mm_paged_attn_workspace_bytes(pa, pb, 4, 1 << 24)
    rc, msg = attend(step=big, rows=1 << 24, ws=4096, ws_bytes=need)
    assert need > 0 and rc == -1 and "grid" in msg
    assert lib.mm_sample_tokens(4096, 4096, 128, 4096, 1 << 22, 100, 1.0, None, 0, None, 0.0, None, 0.0, None, 0, None) == -1


def test_empty_arrays_may_be_null():
    assert append(step=dict(seqs=0, block_table=0, cu_new=0, kv_lens=0))[0] == 0 and attend(step=dict(seqs=0, block_table=0, kv_lens=0))[0] == 0
    assert append(rows=0, k=0, v=0, q=0, q_out=0)[0] == 0


def test_generated_rows_end_with_the_end_token_or_a_failed_draw():
    from multimodal_amd.generation import _trim
    out = torch.tensor([[5, 7, 9, 1], [3, -1, 9, 2], [8, 4, 3, 3], [3, 3, -1, 4]])
    assert [r.tolist() for r in _trim(out, 3)] == [[5, 3], [7, -1], [9, 9, 3], [1, 2, 3]]
    assert [r.tolist() for r in _trim(out, None)] == [[5, 3, 8, 3], [7, -1], [9, 9, 3, -1], [1, 2, 3, 4]]


def test_workspace_of_a_long_chunk_is_not_multiplied_by_the_single_tokens_splits():
    """The few-row form's partial results are kept for at most 16 rows a sequence and key head."""
    lib = _lib.get_lib()
    step = dict(seqs=1, max_new=8192, max_kv=131072, max_pages=8192, table_stride=8192)
    a, b, pa, pb = refs(kv=dict(hn=128, heads=8, page=8 * 16 * 128, head=16 * 128, slot=128), step=step)
    need = lib.mm_paged_attn_workspace_bytes(pa, pb, 32, 8192)
    assert 0 < need <= 32 * 8 * 16 * 130 * 4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_generation_leaves_the_rotary_tables_of_training_alone(dtype):
    """A captured training step reads the tables it was captured with: generation's, of other lengths, are others, and stay too."""
    from multimodal_amd.model.positional_embeddings import RotaryEmbedding
    rot = RotaryEmbedding(16, precision=dtype).to(dtype)
    x = torch.zeros(1, dtype=dtype)
    cos, sin = rot.forward(x, seq_len=64)
    seen = [rot.kept_tables(x, n) for n in (5, 64, 33, 200, 1, 300)]
    assert rot.cos_cached is cos and rot.sin_cached is sin
    for n, (c, s) in zip((5, 64, 33, 200, 1, 300), seen):
        want_c, want_s = rot.tables(x, n)
        assert c.shape == (n, 16) and c.is_contiguous() and torch.equal(c, want_c) and torch.equal(s, want_s)
    assert seen[1][0].data_ptr() == seen[2][0].data_ptr() == rot.kept_tables(x, 40)[0].data_ptr()
    before = rot.kept_tables(x, 40)[0].clone()
    with torch.no_grad():
        rot.inv_freq.mul_(0.5)  # e.g. a loaded checkpoint
    assert not torch.equal(rot.kept_tables(x, 40)[0], before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tables_of_generation_follow_the_frequencies_the_module_holds(dtype):
    """A buffer that takes the place of inv_freq starts counting its versions anew: the tables are still those of what it holds."""
    from multimodal_amd.model.positional_embeddings import RotaryEmbedding
    x = torch.zeros(1, dtype=dtype)

    def agree(rot):
        for got, want in zip(rot.kept_tables(x, 40), rot.tables(x, 40)):
            assert torch.equal(got, want)
        rot.seq_len_cached = None  # `tables` keeps the last length's

    rot = RotaryEmbedding(16, precision=dtype)
    agree(rot)
    first = rot.kept_tables(x, 40)[0]
    copy = first.clone()
    rot.load_state_dict({"inv_freq": 0.5 * rot.inv_freq}, assign=True)
    agree(rot)
    rot.to(torch.bfloat16).float()  # the frequencies have been rounded
    agree(rot)
    rot.precision = torch.float32
    agree(rot)
    rot.precision = dtype
    with torch.inference_mode():
        rot.inv_freq = 0.25 * rot.inv_freq  # no versions are counted in here
        agree(rot)
        rot.inv_freq.mul_(2.0)
        agree(rot)
    assert torch.equal(first, copy)  # a step captured with them goes on reading them


def test_a_wrong_rotation_position_or_scale_exceeds_the_bounds_of_the_wiring_tests():
    """The mistakes are planted in the oracle: more than twice the attention test's bound (2 spreads) and twice the model test's,
    over the rows of the tokens that came singly and over all of them."""
    import generation_harness as G
    for h, heads, part in G.ATTENTION:
        p, d = G.layer_params(h, heads), int(h // heads * part)
        x = torch.randn(119, h, generator=torch.Generator().manual_seed(1)).bfloat16()
        want, spread = G.attention_by_hand(p, heads, d, x)
        for mistake in G.MISTAKES:
            got = G.attention_by_hand(p, heads, d, x, mistake, new=49)[0]
            for rows in (slice(0, 119), slice(70, 119)):
                assert (got - want)[rows].norm() > 2 * 2.0 * spread[rows].norm(), (h, mistake)
    p = G.model_params()
    for s in (21, 27, 50):
        tokens = torch.randint(0, G.MODEL["V"], (s,), generator=torch.Generator().manual_seed(s))
        want = G.model_logits(p, tokens, torch.float32)[-20:]
        bound = 2 * G.off(G.model_logits(p, tokens, torch.bfloat16)[-20:], want) + G.U
        for mistake in G.MISTAKES:
            assert G.off(G.model_logits(p, tokens, torch.float32, mistake, 20)[-20:], want) > 2 * bound, (s, mistake)


def test_outputs_that_overlap_are_refused():
    """Rows 256 elements apart, heads 64 (4 heads of 64), from address 1 << 20; every call here is refused before any launch."""
    lib = _lib.get_lib()
    at = 1 << 20
    far = at + (1 << 16)

    def append(q_out, qo=(256, 64), q=at, qs=(256, 64), k=far, v=2 * far, rows=8):
        a, b, pa, pb = refs()
        return lib.mm_paged_kv_append(pa, pb, k, 256, 64, v, 256, 64, q, *qs, q_out, *qo, 4, rows, 0, 0, 0, 0, 0, None), lib.mm_last_error().decode()

    def attend(out, os=(256, 64), q=at, qs=(256, 64), lse=far, l_row=4, rows=8):
        a, b, pa, pb = refs()
        return lib.mm_paged_attn_fwd(pa, pb, out, *os, lse, l_row, q, *qs, 4, rows, 0.125, 0, 0, None), lib.mm_last_error().decode()

    three = (768, 192)  # a slice of [rows, heads, 3, 64]
    for call in (append, attend):
        for bad, text in [(dict(), "in part"),                                   # q moved by 8 elements
                          (dict(shift=512), "in part"),                          # by a row
                          (dict(shift=-128), "in part"),                         # by a head
                          (dict(strides=three, other=three), "in part"),
                          (dict(shift=2 * 192, strides=three, other=three), "in part"),   # by a head of the fused projection
                          (dict(shift=0, strides=(512, 64)), "in part"),
                          (dict(shift=0, strides=(256, 72)), "itself"),          # the rows reach into each other
                          (dict(shift=0, strides=(0, 64)), "itself"),
                          (dict(shift=0, strides=(256, 56)), "itself"),
                          (dict(shift=0, strides=(64, 64)), "itself")]:
            bad = {"shift": 16, "strides": (256, 64), "other": (256, 64), **bad}
            rc, msg = call(at + bad["shift"], bad["strides"], qs=bad["other"])
            assert rc == -1 and text in msg, (bad, rc, msg)
    for other in ("k", "v"):
        for where in (at, at + 2 * 63, at + 2 * 256 * 7):
            rc, msg = append(at, **{other: where})
            assert rc == -1 and "k or v" in msg, (other, where, msg)
    for lse in (at, at + 2 * 256 * 7 + 2 * 192, far):
        rc, msg = attend(far, lse=lse)
        assert rc == -1 and "lse overlaps" in msg, (lse, msg)
    assert attend(far, lse=2 * far, l_row=3)[0] == -1
