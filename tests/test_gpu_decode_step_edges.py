"""Decode-step operators where their other tests do not go: pools past 2^32
bytes, tensors with strides, the library's own scratch, batches of a cache's own making
under graph capture."""

from __future__ import annotations

import ctypes

import pytest

from test_gpu_prefix import i32, make, randn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dt,n,H,Hkv,T", [("bf16", 20, 32, 8, 1), ("bf16", 3, 16, 8, 1), ("f32", 5, 16, 8, 2), ("f16", 12, 8, 8, 2)])
def test_pages_past_32_bits(ofh, dt, n, H, Hkv, T):
    """Pages at the far end of pools of more than 2^31 elements, and bounds as far
    apart: the same numbers as from pools that hold these pages alone."""
    F, D, size, shared = ofh, 128, 16, 256
    lengths = [shared + T + 5 * b for b in range(n)]
    k, v, table = make(1, dt, [(n, shared)], lengths, Hkv, D, D, size)
    k, v, near = k.cuda(), v.cuda(), torch.from_numpy(table).cuda()
    pages, P = k.shape[0], (1 << 31) // (Hkv * size * D) + 4096
    far = torch.where(near >= 0, near + (P - pages), near)
    big = [torch.empty((P, Hkv, size, D), dtype=k.dtype, device="cuda") for _ in range(2)]
    assert big[0].numel() > 1 << 31
    for b, x in zip(big, (k, v)):
        b[P - pages:] = x
    q, lens = randn(2, (n, H, T, D), dt).cuda(), i32(lengths)
    groups = F.PrefixGroups([(n, shared)], page_size=size)
    assert torch.equal(F.shared_prefix_attention(q, *big, far, lens, groups=groups),
                       F.shared_prefix_attention(q, k, v, near, lens, groups=groups))
    # bounds, selection and attention over what it selects
    bounds = torch.zeros((pages, Hkv, 2, D), dtype=k.dtype, device="cuda")
    stride = (1 << 31) // (P - 1) // 8 * 8 + 8  # elements between pages: the last stand past 2^31
    wide = torch.zeros((P - 1) * max(stride, bounds[0].numel()) + bounds[0].numel(), dtype=k.dtype, device="cuda").as_strided(
        (P, Hkv, 2, D), (max(stride, bounds[0].numel()), 2 * D, D, 1))
    F.page_bounds(k, bounds, near, lens)
    F.page_bounds(big[0], wide, far, lens)
    assert torch.equal(wide[P - pages:], bounds)
    here = F.SelectedAttention(k, v, bounds, near, lens, heads=H, query_tokens=T, pages=7)
    there = F.SelectedAttention(*big, wide, far, lens, heads=H, query_tokens=T, pages=7)
    assert torch.equal(there.select(q), here.select(q)) and torch.equal(there(q), here(q))
    # appending
    rotary = F.Rotary(D)
    rows = [randn(i, (n, h, T, D), dt).cuda() for i, h in ((3, Hkv), (4, Hkv), (5, H))]
    turned = F.cache_append(*rows[:2], k, v, near, lens, rotary, q=rows[2])
    assert torch.equal(F.cache_append(*rows[:2], *big, far, lens, rotary, q=rows[2]), turned)
    assert torch.equal(big[0][P - pages:], k) and torch.equal(big[1][P - pages:], v)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_selection_of_strided_tensors(ofh, dt):
    """Queries of a fused projection, bounds of one of several layers, results into a
    token-major tensor: as from contiguous ones."""
    F, B, H, Hkv, T, D, size = ofh, 3, 8, 2, 3, 64, 16
    lengths = [700, 90, 333]
    k, v, table = make(1, dt, [(1, 0)] * B, lengths, Hkv, D, D, size)
    k, v, table, lens = k.cuda(), v.cuda(), torch.from_numpy(table).cuda(), i32(lengths)
    bounds = torch.zeros((k.shape[0], Hkv, 2, D), dtype=k.dtype, device="cuda")
    F.page_bounds(k, bounds, table, lens)
    q = randn(2, (B, H, T, D), dt).cuda()
    want = F.SelectedAttention(k, v, bounds, table, lens, heads=H, query_tokens=T, pages=9)
    lists, rows = want.select(q), want(q)
    layers = torch.full((k.shape[0], 3, Hkv, 2, D), 7.0, dtype=k.dtype, device="cuda")
    layers[:, 1] = bounds
    fused = torch.zeros((B, T, H + 2 * Hkv, D), dtype=k.dtype, device="cuda")
    fused[:, :, :H] = q.transpose(1, 2)
    odd = torch.zeros((B, T, H, D + 4), dtype=k.dtype, device="cuda")  # rows of 8-byte alignment, for the selection
    odd[..., 4:] = q.transpose(1, 2)
    wide_table = torch.full((B, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide_table[:, :table.shape[1]] = table
    a = F.SelectedAttention(k, v, layers[:, 1], wide_table[:, :table.shape[1]], lens, heads=H, query_tokens=T, pages=9)
    view = fused[:, :, :H].transpose(1, 2)
    assert not view.is_contiguous() and torch.equal(a.select(view), lists)
    out = torch.full((B, T, H, D), 7.0, dtype=k.dtype, device="cuda").transpose(1, 2)
    chosen = torch.full((B, Hkv, T, 9), 77, dtype=torch.int32, device="cuda")
    assert a.select(view, out=chosen) is chosen and torch.equal(chosen, lists)
    assert a(view, selected=chosen, out=out) is out and torch.equal(out, rows)
    assert torch.equal(a.select(odd[..., 4:].transpose(1, 2)), lists)
    if dt != "f32":
        with pytest.raises(F.OfhError, match="16"):  # the attention reads words
            a(odd[..., 4:].transpose(1, 2), selected=lists)


def test_scratch_of_the_library(ofh):
    """C callers without a workspace: the stream's scratch; under capture a call that does
    not fit it is refused, one that does is captured."""
    F = ofh
    n, H, Hkv, D, size = 6, 16, 2, 64, 16
    k, v, table = make(1, "bf16", [(n, 512)], [900] * n, Hkv, D, D, size)
    k, v, table, lens = k.cuda(), v.cuda(), torch.from_numpy(table).cuda(), i32([900, 513, 700, 20, 0, 899])
    q = randn(2, (n, H, 1, D), "bf16").cuda()
    bounds = torch.zeros((k.shape[0], Hkv, 2, D), dtype=k.dtype, device="cuda")
    F.page_bounds(k, bounds, table, lens)
    shared = F.SharedPrefixAttention(k, v, table, lens, groups=[(n, 512)], heads=H)
    chosen = F.SelectedAttention(k, v, bounds, table, lens, heads=H, pages=40)
    assert shared.workspace_bytes > 0 and chosen.select_workspace_bytes > 0
    want = shared(q), chosen.select(q), chosen(q)
    outs = torch.empty_like(want[0]), torch.empty_like(want[1]), torch.empty_like(want[2])
    L = F.lib()
    p, s = F.PagedParams.from_buffer_copy(shared._params), F.SelectParams.from_buffer_copy(chosen._select_params)
    c = F.PagedParams.from_buffer_copy(chosen._params)
    at = [x.data_ptr() for x in (q, k, v)]

    def calls(stream):
        return [L.ofh_shared_prefix_attention_fwd(ctypes.addressof(p), *shared._more, *at, outs[0].data_ptr(), None, 0, stream),
                L.ofh_select_pages(ctypes.addressof(s), at[0], bounds.data_ptr(), outs[1].data_ptr(), None, 0, stream),
                L.ofh_selected_attention_fwd(ctypes.addressof(c), outs[1].data_ptr(), 40, *at, outs[2].data_ptr(), None, 0, stream)]

    assert calls(torch.cuda.current_stream().cuda_stream) == [0, 0, 0]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, want))
    side = torch.cuda.Stream()  # without scratch yet
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        small = calls(side.cuda_stream)
        error = L.ofh_last_error().decode()
        outs[0].zero_()
    assert small == [F.OFH_ERROR_WORKSPACE_TOO_SMALL, F.OFH_ERROR_WORKSPACE_TOO_SMALL, 0] and "workspace too small" in error
    assert calls(side.cuda_stream) == [0, 0, 0]  # makes the stream's scratch
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        assert calls(side.cuda_stream) == [0, 0, 0]
    for i in range(4):
        lens[0] += -1
        q.mul_(0.9)
        for x in outs:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], shared(q)) and torch.equal(outs[1], chosen.select(q)) and torch.equal(outs[2], chosen(q))


def test_scratch_of_a_long_list(ofh):
    """Attention over a list does without its parts where their scratch does not fit a
    capture: the same row up to the order of its sums."""
    F, D, size = ofh, 128, 16
    k, v, table = make(1, "f32", [(1, 0)], [3000], 2, D, D, size)
    k, v, table, lens = k.cuda(), v.cuda(), torch.from_numpy(table).cuda(), i32([3000])
    q = randn(2, (1, 8, 1, D), "f32").cuda()
    bounds = torch.zeros((k.shape[0], 2, 2, D), device="cuda")
    lists = torch.arange(150, dtype=torch.int32, device="cuda").mul(5).div(4, rounding_mode="floor").int().expand(1, 2, 1, 150).contiguous()
    make_it = lambda splits: F.SelectedAttention(k, v, bounds, table, lens, heads=8, pages=150, max_key_splits=splits)
    a = make_it(0)
    assert a.workspace_bytes > 0 and make_it(1).workspace_bytes == 0
    want, alone = a(q, selected=lists), make_it(1)(q, selected=lists)
    out = torch.empty_like(want)
    p = F.PagedParams.from_buffer_copy(a._params)
    args = [ctypes.addressof(p), lists.data_ptr(), 150, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), None, 0]
    for warm, expected in ((False, alone), (True, want)):
        side = torch.cuda.Stream()
        if warm:
            F.check(F.lib().ofh_selected_attention_fwd(*args, side.cuda_stream))
            side.synchronize()
            assert torch.equal(out, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            F.check(F.lib().ofh_selected_attention_fwd(*args, side.cuda_stream))
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, expected)


def test_a_batch_under_capture(ofh):
    """A layer of a decode step through a cache's batch, captured once and replayed with
    other rows and lengths: append, bounds, shared and selected attention."""
    from onednn_flash_cache import PagedCache
    F = ofh
    cache = PagedCache(layers=1, num_pages=200, page_size=16, kv_heads=2, head_dim=64, bounds=True)
    rotary = F.Rotary(64)
    root = cache.add()
    k, q = (randn(i, (1, h, 200, 64), "bf16").cuda() for i, h in enumerate((2, 8)))
    cache.extend([root], [200]).append(0, k, k, rotary, q)
    seqs = [root] + [cache.fork(root) for _ in range(3)]
    batch = cache.extend(seqs, [16] * 4)  # (room for the steps)
    batch.counts.fill_(1)
    k, v, q = (randn(5 + i, (4, h, 16, 64), "bf16").cuda() for i, h in enumerate((2, 2, 8)))
    q1 = q[:, :, :1].contiguous()

    def layer():
        turned = batch.append(0, k, v, rotary, q)
        return turned, batch.attend_shared(0, q1), batch.attend_selected(0, q1, pages=5)

    batch.lengths.fill_(201)
    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = layer()
    for step in range(4):
        batch.lengths.fill_(202 + 3 * step)
        for i, x in enumerate((k, v, q1)):
            x.copy_(randn(20 + 3 * step + i, x.shape, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs]
        kept = cache.k_pages.clone(), cache.v_pages.clone(), cache.k_bounds.clone()
        assert all(torch.equal(x, y) for x, y in zip(got, layer()))
        assert all(torch.equal(x, y) for x, y in zip(kept, (cache.k_pages, cache.v_pages, cache.k_bounds)))
