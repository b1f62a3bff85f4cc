"""GPU tests of the 8-bit KV cache operators: codes and exponents bit for bit against a plain quantiser, attention
against 64 bits within bounds derived in q8_ref.attention, and the four operators together."""
import numpy as np
import pytest
import torch

from tests import q8_ref as R

pytestmark = pytest.mark.gpu

FP16, BF16, D = 4, 5, 128


@pytest.fixture(scope="module")
def ops():
    from llm_simple_b200 import ops as o
    o.lib()
    return o


@pytest.fixture(autouse=True)
def _status(request):
    """Every test starts and, unless it says otherwise, ends with the status word at 0."""
    from llm_simple_b200 import ops as o
    torch.cuda.synchronize()
    o.gpu_ops_clear_kernel_status()
    yield
    torch.cuda.synchronize()
    if "bad" not in request.node.name:
        assert o.gpu_ops_kernel_status() == 0
    o.gpu_ops_clear_kernel_status()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def _randn(shape, dt, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(R.TORCH_DT[dt])


def _np32(t):
    return t.float().cpu().numpy()


LAYOUTS = [("head", 0), ("token", 0), ("paged", 64), ("paged", 256)]


# ------------------------------------------------------------------------------------------ write and read
@pytest.mark.parametrize("layout,page", LAYOUTS)
@pytest.mark.parametrize("dt,neox", [(FP16, False), (BF16, True)])
def test_append_then_read(ops, dt, neox, layout, page):
    H, kvH, max_pos = 6, 2, 700
    new, start = [1, 0, 65, 300, 7, 0], [699, 5, 63, 100, 0, 0]
    B, total, extra = len(new), sum(new), 3
    c = R.Cache(ops, dt, B, H, kvH, max_pos, layout, page, neox, seed=2)
    q, k, v = (_randn((total + extra, h, D), dt, s, 2.0) for h, s in ((H, 1), (kvH, 2), (kvH, 3)))
    tab = R.rope_table(max_pos)
    q_out = torch.full_like(q, 7.0)
    before = [t.clone() for t in (c.k, c.kx, c.v, c.vx)]
    tok = _starts(new)
    tok_d, start_d, tab_d = _i32(tok), _i32(start), torch.from_numpy(tab).cuda()
    ops.gpu_rope_kv_append_q8_layer(c.desc, c.pages, c.kv, q_out, q, k, v, tab_d, tok_d, start_d, total + extra)
    torch.cuda.synchronize()
    assert bool((q_out[total:] == 7.0).all())                     # rows behind the last sequence
    expect = R.Cache(ops, dt, B, H, kvH, max_pos, layout, page, neox, seed=2)
    k_back, v_back = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    for b in range(B):
        rows = slice(tok[b], tok[b + 1])
        pos = np.arange(start[b], start[b] + new[b])
        if not new[b]:
            continue
        want_q = torch.from_numpy(R.rotate_f32(_np32(q[rows]), tab[pos], neox)).to(R.TORCH_DT[dt]).cuda()
        assert torch.equal(q_out[rows], want_q)
        expect.put(b, pos, *R.quantise(R.rotate_f32(_np32(k[rows]), tab[pos], neox)), *R.quantise(_np32(v[rows])))
    for got, want, old, name in zip((c.k, c.kx, c.v, c.vx), (expect.k, expect.kx, expect.v, expect.vx), before, "k kx v vx".split()):
        assert torch.equal(got, want), name                       # what was written, bit for bit, and nothing else
        assert not torch.equal(got, old)
    ops.gpu_kv_read_q8_layer(c.desc, c.pages, c.kv, k_back, v_back, tok_d, start_d, total + extra)
    torch.cuda.synchronize()
    assert bool((k_back[total:] == 7.0).all()) and bool((v_back[total:] == 7.0).all())
    for b in range(B):
        if new[b]:
            kc, kx, vc, vx = c.rows(b, np.arange(start[b], start[b] + new[b]))
            rows = slice(tok[b], tok[b + 1])
            assert torch.equal(k_back[rows], R.values(kc, kx).to(k.dtype))
            assert torch.equal(v_back[rows], R.values(vc, vx).to(k.dtype))


@pytest.mark.parametrize("batch", [1, 7, 8, 9, 64, 65, 600])
def test_rows_find_their_sequence(ops, batch):
    """Many sequences, most of them with no or one token: every row lands where a plain loop puts it."""
    rng = np.random.default_rng(batch)
    new = rng.choice([0, 0, 1, 1, 2, 5], batch)
    new[batch // 2] = 3
    start = rng.integers(0, 10, batch)
    c = R.Cache(ops, BF16, batch, 1, 1, 16, "head")
    total = int(new.sum())
    k, v = _randn((total, 1, D), BF16, 5), _randn((total, 1, D), BF16, 6)
    tab = torch.from_numpy(R.rope_table(16)).cuda()
    ops.gpu_rope_kv_append_q8_layer(c.desc, None, c.kv, None, None, k, v, tab, _i32(_starts(new)), _i32(start), total)
    torch.cuda.synchronize()
    vc, vx = R.quantise(_np32(v))
    t = 0
    for b in range(batch):
        for r in range(new[b]):
            assert np.array_equal(c.v[b, 0, start[b] + r].cpu().numpy(), vc[t, 0])
            assert int(c.vx[b, 0, start[b] + r]) == vx[t, 0]
            t += 1
    assert int((c.vx != 255).sum()) == total


@pytest.mark.parametrize("dt", [FP16, BF16])
def test_rows_of_special_values(ops, dt):
    """Zeros, the smallest and largest magnitudes, every border between two exponents, and values that are not finite."""
    t = R.TORCH_DT[dt]
    fi = torch.finfo(t)
    ramp = torch.linspace(-1, 1, D)
    rows = [torch.zeros(D), -torch.zeros(D), ramp * 448, ramp * 449, ramp * 450, ramp * fi.max, ramp * fi.tiny, ramp * 2.0 ** -14 * 1.75,
            torch.full((D,), fi.smallest_normal), torch.full((D,), -fi.max), ramp * 2.0 ** -6, torch.arange(D) * 2.0 ** -9]
    for bad in (float("inf"), -float("inf"), float("nan")):
        x = ramp.clone()
        x[17] = bad
        rows.append(x)
    v = torch.stack(rows)[:, None].to(t).cuda().contiguous()
    n = v.shape[0]
    c = R.Cache(ops, dt, 1, 1, 1, 64, "head")
    tab = torch.zeros(64, 64, 2, device="cuda")
    tab[..., 0] = 1.0                                            # no rotation: K is quantised as it is
    ops.gpu_rope_kv_append_q8_layer(c.desc, None, c.kv, None, None, v, v, tab, _i32([0, n]), _i32([0]), n)
    back_k, back_v = torch.empty_like(v), torch.empty_like(v)
    ops.gpu_kv_read_q8_layer(c.desc, None, c.kv, back_k, back_v, _i32([0, n]), None, n)
    torch.cuda.synchronize()
    codes, exps = R.quantise(_np32(v))
    assert np.array_equal(c.vx[0, 0, :n].cpu().numpy(), exps[:, 0])
    assert np.array_equal(c.v[0, 0, :n].cpu().numpy(), codes[:, 0])
    assert np.array_equal(c.kx[0, 0, :n].cpu().numpy(), exps[:, 0])
    finite = exps[:, 0] != 255
    assert bool(torch.isnan(back_v[~torch.from_numpy(finite)]).all()) and int(finite.sum()) == n - 3
    want = R.values(c.v[0, 0, :n][:, None], c.vx[0, 0, :n][:, None]).to(t)
    assert torch.equal(back_v[torch.from_numpy(finite)], want[torch.from_numpy(finite)])


def test_append_from_a_fused_row_in_place(ops):
    """q, k and v are columns of one projection row; q is rotated in place; only one of the two outputs is read."""
    H, kvH, n, width = 4, 2, 70, (4 + 2 * 2) * D + 64
    row = _randn((n, width), BF16, 9)
    keep = row.clone()
    c = R.Cache(ops, BF16, 1, H, kvH, 128, "paged", 64, True)
    c.desc.q_tok_stride = c.desc.kv_in_tok_stride = width
    tab = R.rope_table(128)
    q, k, v = row[:, :H * D], row[:, H * D:(H + kvH) * D], row[:, (H + kvH) * D:(H + 2 * kvH) * D]
    ops.gpu_rope_kv_append_q8_layer(c.desc, c.pages, c.kv, q, q, k, v, torch.from_numpy(tab).cuda(), _i32([0, n]), _i32([11]), n)
    torch.cuda.synchronize()
    pos = np.arange(11, 11 + n)
    want = R.rotate_f32(_np32(keep[:, :H * D].reshape(n, H, D)), tab[pos], True)
    assert torch.equal(row[:, :H * D], torch.from_numpy(want).to(row.dtype).cuda().reshape(n, H * D))
    assert torch.equal(row[:, H * D:], keep[:, H * D:])
    codes, exps = R.quantise(_np32(keep[:, (H + kvH) * D:(H + 2 * kvH) * D].reshape(n, kvH, D)))
    assert np.array_equal(c.rows(0, pos)[2].cpu().numpy(), codes)
    only_v = torch.zeros((n, width), dtype=row.dtype, device="cuda")
    ops.gpu_kv_read_q8_layer(c.desc, c.pages, c.kv, None, only_v, _i32([0, n]), _i32([11]), n)
    torch.cuda.synchronize()
    assert torch.equal(only_v[:, :kvH * D].reshape(n, kvH, D), R.values(*c.rows(0, pos)[2:]).to(row.dtype))
    assert not bool(only_v[:, kvH * D:].any())


def test_bad_positions_and_pages_are_skipped_and_reported(ops):
    c = R.Cache(ops, BF16, 3, 2, 1, 100, "paged", 64)
    c.table[1, 0], c.table[2, 1] = -1, 10 ** 6
    before = [t.clone() for t in (c.k, c.v, c.kx, c.vx)]
    k = _randn((6, 1, D), BF16, 1)
    q = _randn((6, 2, D), BF16, 2)
    q_out = torch.zeros_like(q)
    tab = torch.from_numpy(R.rope_table(100)).cuda()
    # sequence 0: positions 99 (fine) and 100 (beyond); 1: page -1; 2: page 10^6 and a negative position
    tok, start = _i32([0, 2, 4, 6]), _i32([99, 0, 64])
    ops.gpu_rope_kv_append_q8_layer(c.desc, c.pages, c.kv, q_out, q, k, k, tab, tok, start, 6)
    torch.cuda.synchronize()
    assert ops.gpu_ops_kernel_status() == 41
    ops.gpu_ops_clear_kernel_status()
    assert int((c.kx != before[2]).sum()) == 1 and int((c.vx != before[3]).sum()) == 1
    assert not bool(q_out[1].any()) and bool(q_out[0].any()) and bool(q_out[2].any())
    ops.gpu_rope_kv_append_q8_layer(c.desc, c.pages, c.kv, None, None, k, k, tab, _i32([0, 0, 0, 2]), _i32([0, 0, -2]), 6)
    back = torch.full((6, 1, D), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.gpu_kv_read_q8_layer(c.desc, c.pages, c.kv, back, None, tok, start, 6)
    torch.cuda.synchronize()
    assert ops.gpu_ops_kernel_status() == 41
    assert bool((back[1:] == 3.0).all()) and not bool((back[0] == 3.0).all())
    assert int((c.kx != before[2]).sum()) == 1


def test_offsets_beyond_32_bits(ops):
    """A flat cache whose second sequence starts 2.3 GB in: every operator reaches it."""
    H, kvH, n = 2, 1, 70
    c = R.Cache(ops, FP16, 2, H, kvH, 128, "head")
    stride = (1 << 31) + (1 << 28)
    big_k, big_v = (torch.empty(stride + 128 * D, dtype=torch.uint8, device="cuda") for _ in range(2))
    small = R.Cache(ops, FP16, 2, H, kvH, 128, "head")
    c.desc.cache_seq_stride = stride
    c.kv.k, c.kv.v = big_k.data_ptr(), big_v.data_ptr()
    k, v, q = _randn((n, kvH, D), FP16, 1), _randn((n, kvH, D), FP16, 2), _randn((n, H, D), FP16, 3)
    tab = torch.from_numpy(R.rope_table(128)).cuda()
    tok, start = _i32([0, 0, n]), _i32([0, 0])
    outs = []
    for x in (c, small):
        qo, o, kb, vb, od = (torch.zeros_like(t) for t in (q, q, k, v, q[:2]))
        ops.gpu_rope_kv_append_q8_layer(x.desc, None, x.kv, qo, q, k, v, tab, tok, start, n)
        nb = ops.gpu_attn_chunk_q8_workspace_bytes(x.desc, n, n, n)
        ws = torch.empty(max(16, nb), dtype=torch.uint8, device="cuda")
        ops.gpu_attn_chunk_q8_layer(x.desc, None, x.kv, o, qo, tok, start, n, n, n, 0, 0, ws, nb)
        nb = ops.gpu_attn_decode_q8_workspace_bytes(x.desc, n)
        ws = torch.empty(max(16, nb), dtype=torch.uint8, device="cuda")
        ops.gpu_attn_decode_q8_layer(x.desc, None, x.kv, od, qo[:2], _i32([0, n]), n, 0, 0, ws, nb)
        ops.gpu_kv_read_q8_layer(x.desc, None, x.kv, kb, vb, tok, None, n)
        torch.cuda.synchronize()
        outs.append((o, od, kb, vb))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(a.any())


def test_tensors_of_another_device_are_refused(ops):
    c = R.Cache(ops, FP16, 1, 2, 1, 64, "head")
    x = torch.zeros((1, 2, D), dtype=torch.float16)              # in host memory: its address must not reach a kernel
    with pytest.raises(ops.GpuOpsError, match="cpu"):
        ops.gpu_attn_decode_q8_layer(c.desc, None, c.kv, x.cuda(), x, _i32([0]), 1, 0, 0, None, 0)
    with pytest.raises(ops.GpuOpsError, match="cpu"):
        ops.gpu_kv_read_q8_layer(c.desc, None, c.kv, x, None, _i32([0, 1]), None, 1)
    with pytest.raises(ops.GpuOpsError, match="cpu"):
        ops.gpu_rope_kv_append_q8_layer(c.desc, None, c.kv, None, None, x.cuda(), x.cuda(), x, _i32([0, 1]), _i32([0]), 1)
    with pytest.raises(ops.GpuOpsError, match="cpu"):
        ops.gpu_attn_chunk_q8_layer(c.desc, None, c.kv, x.cuda(), x.cuda(), torch.zeros(2, dtype=torch.int32), _i32([0]), 1, 1, 1, 0, 0, None, 0)


# ------------------------------------------------------------------------------------------ decode
def _decode(ops, c, q, lens, mx=None, window=0, sink=0, out=None):
    mx = mx or max(1, max(lens))
    out = torch.full_like(q, 7.0) if out is None else out
    n = ops.gpu_attn_decode_q8_workspace_bytes(c.desc, mx)
    ws = torch.full((max(16, n),), 0xFF, dtype=torch.uint8, device="cuda")
    ops.gpu_attn_decode_q8_layer(c.desc, c.pages, c.kv, out, q, _i32(lens), mx, window, sink, ws, n)
    torch.cuda.synchronize()
    return out


def _check_decode(c, q, out, lens, window, sink, what):
    for b, n in enumerate(lens):
        want, tol = R.attention(c, q[b:b + 1], b, [n - 1], window, sink, R.half_step(c.dt))
        R.assert_close(out[b:b + 1], want, tol, "%s, sequence %d of %d positions" % (what, b, n))


@pytest.mark.parametrize("layout,page", LAYOUTS)
@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("window,sink", [(0, 0), (100, 0), (64, 4), (1, 0), (129, 70), (5000, 3)])
def test_decode(ops, layout, page, dt, window, sink):
    H, kvH = 10, 2
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700, 1023]
    c = R.Cache(ops, dt, len(lens), H, kvH, 1100, layout, page, seed=4)
    c.fill(lens)
    q = _randn((len(lens), H, D), dt, 3)
    _check_decode(c, q, _decode(ops, c, q, lens, 1100, window, sink), lens, window, sink, "decode")


@pytest.mark.parametrize("H,kvH", [(1, 1), (4, 4), (12, 2), (28, 4), (8, 1), (16, 1), (32, 2)])
def test_decode_head_groups(ops, H, kvH):
    lens = [300, 77]
    c = R.Cache(ops, BF16, 2, H, kvH, 320, "paged", 64)
    c.fill(lens)
    q = _randn((2, H, D), BF16, 3, 3.0)
    _check_decode(c, q, _decode(ops, c, q, lens), lens, 0, 0, "decode")


@pytest.mark.parametrize("batch,kvH,n", [(1, 1, 20000), (1, 8, 9000), (3, 2, 6000), (40, 8, 600)])
def test_decode_long(ops, batch, kvH, n):
    """Few and many sequences of very different lengths: the cache is split over the GPU in different ways."""
    lens = [n] + [int(n * (0.1 + 0.8 * ((b * 0.618) % 1))) for b in range(1, batch)]
    c = R.Cache(ops, FP16, batch, 4 * kvH, kvH, n, "paged", 128)
    c.fill(lens)
    q = _randn((batch, 4 * kvH, D), FP16, 3)
    out = _decode(ops, c, q, lens)
    for b in sorted({0, 1, batch // 2, batch - 1} & set(range(batch))):
        want, tol = R.attention(c, q[b:b + 1], b, [lens[b] - 1], 0, 0, R.half_step(FP16))
        R.assert_close(out[b:b + 1], want, tol, "sequence %d" % b)
    for _ in range(10):
        assert torch.equal(out, _decode(ops, c, q, lens))        # the same bits every time


def test_decode_unseen_pages_need_not_exist(ops):
    """Pages without a visible position may be given back: their table entries are not read."""
    lens, window, sink = [1000, 640, 70], 200, 4
    c = R.Cache(ops, BF16, 3, 4, 2, 1024, "paged", 64)
    c.fill(lens)
    q = _randn((3, 4, D), BF16, 3)
    first = _decode(ops, c, q, lens, 1024, window, sink)
    for b, n in enumerate(lens):
        for page in range(c.table.shape[1]):
            lo, hi = page * 64, page * 64 + 64
            if hi <= n - window and lo >= sink or lo >= n:
                c.table[b, page] = -12345
    _check_decode(c, q, first, lens, window, sink, "decode")
    assert torch.equal(first, _decode(ops, c, q, lens, 1024, window, sink))


def test_decode_rows_that_are_not_finite(ops):
    """A poisoned position makes the rows that see it NaN, in its head only; behind a window it does nothing."""
    lens = [300, 300, 300]
    c = R.Cache(ops, BF16, 3, 4, 2, 320, "head")
    c.fill(lens)
    c.kx[0, 1, 150] = 255
    c.vx[1, 0, 290] = 255
    c.vx[2, 0, 90] = 255
    q = _randn((3, 4, D), BF16, 3)
    out = _decode(ops, c, q, lens, 320)
    _check_decode(c, q, out, lens, 0, 0, "decode")
    assert bool(torch.isnan(out[0, 2:]).all()) and not bool(torch.isnan(out[0, :2]).any())
    out = _decode(ops, c, q, lens, 320, 100, 0)
    _check_decode(c, q, out, lens, 100, 0, "decode")
    assert not bool(torch.isnan(out[2]).any())
    q[1, 1, 5] = float("inf")                                    # a query row that is not finite spoils itself alone
    out = _decode(ops, c, q, lens, 320, 100, 0)
    assert bool(torch.isnan(out[1, 1]).all()) and not bool(torch.isnan(out[2]).any()) and not bool(torch.isnan(out[0]).any())


def test_decode_strided_rows(ops):
    lens, H = [130, 5], 4
    c = R.Cache(ops, FP16, 2, H, 2, 256, "paged", 128)
    c.fill(lens)
    wide, out = _randn((2, 2 * H * D), FP16, 3), torch.zeros((2, H * D + 72), dtype=torch.float16, device="cuda")
    c.desc.q_seq_stride, c.desc.out_seq_stride = wide.stride(0), out.stride(0)
    _decode(ops, c, wide, lens, out=out)
    _check_decode(c, wide[:, :H * D].reshape(2, H, D), out[:, :H * D].reshape(2, H, D), lens, 0, 0, "decode")
    assert not bool(out[:, H * D:].any())


@pytest.mark.parametrize("scale_k,scale_v", [(1e-30, 1.0), (1.0, 1e-28), (3e4, 1e30), (1.0, 3e33)])
def test_decode_extreme_magnitudes(ops, scale_k, scale_v):
    """Exponents far from 0 neither overflow nor vanish on the way."""
    n = 200
    c = R.Cache(ops, BF16, 1, 2, 1, 256, "head")
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((n, 1, D)) * scale_k, rng.standard_normal((n, 1, D)) * scale_v
    c.put(0, np.arange(n), *R.quantise(k), *R.quantise(v))
    q = _randn((1, 2, D), BF16, 3, 1e-3 if scale_k > 1 else 1.0)
    _check_decode(c, q, _decode(ops, c, q, [n]), [n], 0, 0, "decode")


def test_decode_bad_lengths_are_reported(ops):
    c = R.Cache(ops, BF16, 2, 2, 1, 128, "head")
    c.fill([128, 50])
    q = _randn((2, 2, D), BF16, 3)
    out = _decode(ops, c, q, [128, 50], 100)                     # the bound is understated
    assert ops.gpu_ops_kernel_status() == 40
    want, tol = R.attention(c, q[1:], 1, [49], 0, 0, R.half_step(BF16))
    R.assert_close(out[1:], want, tol)
    ops.gpu_ops_clear_kernel_status()
    out = _decode(ops, c, q, [-5, 50], 100)                      # a negative length is an empty cache
    assert ops.gpu_ops_kernel_status() == 0 and not bool(out[0].any())


def test_decode_captured_and_replayed(ops):
    """A graph captured once is replayed with other lengths, another table and other rows in the cache."""
    lens = [100, 400]
    c = R.Cache(ops, BF16, 2, 4, 2, 512, "paged", 64)
    c.fill([512, 512])
    q = _randn((2, 4, D), BF16, 3)
    lens_d, out = _i32(lens), torch.zeros_like(q)
    n = ops.gpu_attn_decode_q8_workspace_bytes(c.desc, 512)
    ws = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")

    def call():
        ops.gpu_attn_decode_q8_layer(c.desc, c.pages, c.kv, out, q, lens_d, 512, 0, 0, ws, n)

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens in ([100, 400], [512, 1], [0, 65]):
        lens_d.copy_(_i32(lens))
        out.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        _check_decode(c, q, out, lens, 0, 0, "replay")


# ------------------------------------------------------------------------------------------ chunks
def _chunk(ops, c, q, new, start, window=0, sink=0, out=None, max_new=None, mx=None):
    total = q.shape[0]
    max_new = max_new or max(1, max(new))
    mx = mx or max(1, max(s + n for s, n in zip(start, new)))
    out = torch.full_like(q, 7.0) if out is None else out
    n = ops.gpu_attn_chunk_q8_workspace_bytes(c.desc, total, max_new, mx)
    ws = torch.full((max(16, n),), 0xFF, dtype=torch.uint8, device="cuda")
    ops.gpu_attn_chunk_q8_layer(c.desc, c.pages, c.kv, out, q, _i32(_starts(new)), _i32(start), total, max_new, mx, window, sink,
                                ws, n)
    torch.cuda.synchronize()
    return out


def _check_chunk(c, q, out, new, start, window, sink, what="chunk"):
    tok = _starts(new)
    for b, n in enumerate(new):
        if not n:
            continue
        rows = slice(tok[b], tok[b + 1])
        want, tol = R.attention(c, q[rows], b, list(range(start[b], start[b] + n)), window, sink, R.half_step(c.dt))
        R.assert_close(out[rows], want, tol, "%s, sequence %d: %d rows behind %d positions" % (what, b, n, start[b]))
    assert bool((out[tok[-1]:] == 7.0).all())                    # rows behind the last sequence


@pytest.mark.parametrize("layout,page", LAYOUTS)
@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("window,sink", [(0, 0), (100, 0), (64, 4), (1, 0), (129, 140)])
def test_chunk(ops, layout, page, dt, window, sink):
    H, kvH = 10, 2
    new, start = [1, 0, 130, 64, 17, 257, 3], [0, 9, 0, 127, 511, 300, 700]
    c = R.Cache(ops, dt, len(new), H, kvH, 800, layout, page, seed=4)
    c.fill([s + n for s, n in zip(start, new)])
    q = _randn((sum(new) + 2, H, D), dt, 3)
    _check_chunk(c, q, _chunk(ops, c, q, new, start, window, sink), new, start, window, sink)


@pytest.mark.parametrize("H,kvH", [(1, 1), (4, 4), (12, 2), (28, 4), (8, 1), (16, 1), (32, 2)])
def test_chunk_head_groups(ops, H, kvH):
    new, start = [70, 40], [150, 0]
    c = R.Cache(ops, BF16, 2, H, kvH, 320, "paged", 64)
    c.fill([220, 40])
    q = _randn((110, H, D), BF16, 3, 2.0)
    _check_chunk(c, q, _chunk(ops, c, q, new, start), new, start, 0, 0)


@pytest.mark.parametrize("new,start", [([1], [5000]), ([3, 2, 3], [1000, 0, 40]), ([40], [6000]), ([600], [0]), ([1, 500, 1, 2], [3000, 10, 0, 90])])
@pytest.mark.parametrize("window,sink", [(0, 0), (300, 4)])
def test_chunk_few_rows_and_long_caches(ops, new, start, window, sink):
    """Drafts, short chunks behind long prefixes, prompts, and batches of all of these."""
    H, kvH = 8, 2
    c = R.Cache(ops, FP16, len(new), H, kvH, 6100, "paged", 64)
    c.fill([s + n for s, n in zip(start, new)])
    q = _randn((sum(new), H, D), FP16, 3)
    out = _chunk(ops, c, q, new, start, window, sink)
    _check_chunk(c, q, out, new, start, window, sink)
    assert torch.equal(out, _chunk(ops, c, q, new, start, window, sink))


@pytest.mark.parametrize("window,sink", [(0, 0), (500, 4)])
def test_chunk_many_blocks_per_cta(ops, window, sink):
    """More blocks than CTAs, some of them with rows in the first of their two tiles only (and few tiles of the cache),
    so that a CTA goes through many pieces."""
    H, kvH = 40, 8
    new = [33, 400, 21, 1, 230, 5, 50, 60] * 4
    start = [(b * 379) % 1100 for b in range(len(new))]
    c = R.Cache(ops, FP16, len(new), H, kvH, 1600, "paged", 128)
    c.fill([s + n for s, n in zip(start, new)])
    q = _randn((sum(new), H, D), FP16, 3)
    out = _chunk(ops, c, q, new, start, window, sink)
    _check_chunk(c, q, out, new, start, window, sink)
    assert torch.equal(out, _chunk(ops, c, q, new, start, window, sink))


def test_chunk_unseen_pages_need_not_exist(ops):
    new, start, window, sink = [140, 5], [800, 300], 150, 4
    c = R.Cache(ops, BF16, 2, 4, 2, 1024, "paged", 64)
    c.fill([940, 305])
    q = _randn((145, 4, D), BF16, 3)
    first = _chunk(ops, c, q, new, start, window, sink)
    _check_chunk(c, q, first, new, start, window, sink)
    for b in range(2):
        for page in range(c.table.shape[1]):
            lo, hi = page * 64, page * 64 + 64
            if (hi <= start[b] - window + 1 and lo >= sink) or lo >= start[b] + new[b]:
                c.table[b, page] = 1 << 30
    assert torch.equal(first, _chunk(ops, c, q, new, start, window, sink))


def test_chunk_rows_that_are_not_finite(ops):
    new, start = [200, 150], [100, 0]
    c = R.Cache(ops, FP16, 2, 4, 2, 320, "paged", 128)
    c.fill([300, 150])
    q = _randn((350, 4, D), FP16, 3)
    kc, kx, vc, vx = (t.clone() for t in c.rows(0, np.arange(300)))
    kx[250, 0] = 255                                             # seen by the last fifty rows of sequence 0, KV head 0
    vx[20, 1] = 255                                              # seen by all rows of KV head 1
    c.put(0, np.arange(300), *(t.cpu().numpy() for t in (kc, kx, vc, vx)))
    out = _chunk(ops, c, q, new, start)
    _check_chunk(c, q, out, new, start, 0, 0)
    assert int(torch.isnan(out[:200, 0, 0]).sum()) == 50 and bool(torch.isnan(out[:200, 2]).all()) and not bool(torch.isnan(out[200:]).any())
    _check_chunk(c, q, _chunk(ops, c, q, new, start, 60, 0), new, start, 60, 0)
    q[7, 3, 100] = float("nan")                                  # a query row that is not finite spoils itself alone
    out = _chunk(ops, c, q, new, start, 60, 0)
    assert bool(torch.isnan(out[7, 3]).all()) and not bool(torch.isnan(out[6, 3]).any()) and not bool(torch.isnan(out[8, 3]).any())


@pytest.mark.parametrize("gap", [2.0 ** 6, 2.0 ** 18])
def test_chunk_tokens_of_very_different_size(ops, gap):
    """Rows far apart in magnitude inside one tile keep their own precision (all of them are exact in the product up
    to a gap of 2^22)."""
    n = 256
    c = R.Cache(ops, BF16, 1, 2, 1, 256, "head")
    rng = np.random.default_rng(0)
    size = np.where(np.arange(n) % 7 == 3, gap, 1.0)[:, None, None]
    k, v = rng.standard_normal((n, 1, D)) / size, rng.standard_normal((n, 1, D)) * size
    c.put(0, np.arange(n), *R.quantise(k), *R.quantise(v))
    q = _randn((n, 2, D), BF16, 3)
    _check_chunk(c, q, _chunk(ops, c, q, [n], [0], 40, 0), [n], [0], 40, 0)


@pytest.mark.parametrize("scale_k,scale_v", [(1e-30, 1.0), (1.0, 1e-28), (3e4, 1e30), (1.0, 3e33)])
def test_chunk_extreme_magnitudes(ops, scale_k, scale_v):
    n = 200
    c = R.Cache(ops, BF16, 1, 2, 1, 256, "head")
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((n, 1, D)) * scale_k, rng.standard_normal((n, 1, D)) * scale_v
    c.put(0, np.arange(n), *R.quantise(k), *R.quantise(v))
    q = _randn((60, 2, D), BF16, 3, 1e-3 if scale_k > 1 else 1.0)
    _check_chunk(c, q, _chunk(ops, c, q, [60], [n - 60]), [60], [n - 60], 0, 0)


def test_chunk_strided_rows(ops):
    new, start, H = [100, 30], [5, 0], 4
    c = R.Cache(ops, FP16, 2, H, 2, 256, "token")
    c.fill([105, 30])
    wide, out = _randn((130, 2 * H * D), FP16, 3), torch.zeros((130, H * D + 72), dtype=torch.float16, device="cuda")
    c.desc.q_tok_stride, c.desc.out_tok_stride = wide.stride(0), out.stride(0)
    _chunk(ops, c, wide, new, start, out=out)
    _check_chunk(c, wide[:, :H * D].reshape(130, H, D), out[:, :H * D].reshape(130, H, D), new, start, 0, 0)
    assert not bool(out[:, H * D:].any())


def test_chunk_bad_bounds_are_reported(ops):
    """An understated bound, a position beyond the cache, a page outside the pool: a status, and the other sequences
    keep their results."""
    new, start = [40, 33], [80, 10]
    for kind in ("max_new", "max_kv_len", "position", "page"):
        c = R.Cache(ops, BF16, 2, 4, 2, 128, "paged", 64)
        c.fill([120, 43])
        q = _randn((73, 4, D), BF16, 3)
        st = list(start)
        if kind == "page":
            c.table[0, 1] = 77777
        if kind == "position":
            st[0] = 120
        out = _chunk(ops, c, q, new, st, max_new=33 if kind == "max_new" else None, mx={"max_kv_len": 60, "position": 128}.get(kind))
        got = ops.gpu_ops_kernel_status()
        assert got in ((0, 40) if kind == "max_new" else (40,) if kind == "max_kv_len" else (41,)), (kind, got)
        ops.gpu_ops_clear_kernel_status()
        want, tol = R.attention(c, q[40:], 1, list(range(10, 43)), 0, 0, R.half_step(BF16))
        R.assert_close(out[40:], want, tol, kind)


def test_chunk_bad_rows_are_reported(ops):
    """Positions before the cache see nothing; rows whose starts decrease are not computed."""
    c = R.Cache(ops, BF16, 2, 4, 2, 128, "paged", 64)
    c.fill([128, 43])
    q = _randn((73, 4, D), BF16, 3)
    out = _chunk(ops, c, q, [40, 33], [-3, 10], mx=128)
    assert ops.gpu_ops_kernel_status() == 41
    ops.gpu_ops_clear_kernel_status()
    assert not bool(out[:3].any())
    for b, rows, pos in ((0, slice(3, 40), range(37)), (1, slice(40, 73), range(10, 43))):
        want, tol = R.attention(c, q[rows], b, list(pos), 0, 0, R.half_step(BF16))
        R.assert_close(out[rows], want, tol)
    for max_new in (40, 4):                                      # the tcgen05 kernel, and the one for few rows
        n = ops.gpu_attn_chunk_q8_workspace_bytes(c.desc, 73, max_new, 128)
        ws = torch.full((max(16, n),), 0xFF, dtype=torch.uint8, device="cuda")
        out = torch.full_like(q, 7.0)
        ops.gpu_attn_chunk_q8_layer(c.desc, c.pages, c.kv, out, q, _i32([0, 60, 20]), _i32([0, 0]), 73, max_new, 128, 0, 0, ws, n)
        torch.cuda.synchronize()
        assert ops.gpu_ops_kernel_status() in (40, 41)
        assert bool((out[60:] == 7.0).all())
        ops.gpu_ops_clear_kernel_status()


def test_chunk_captured_and_replayed(ops):
    c = R.Cache(ops, BF16, 3, 4, 2, 512, "paged", 64)
    c.fill([512] * 3)
    q = _randn((200, 4, D), BF16, 3)
    tok, start, out = _i32([0, 0, 0, 0]), _i32([0, 0, 0]), torch.zeros_like(q)
    n = ops.gpu_attn_chunk_q8_workspace_bytes(c.desc, 200, 200, 512)
    ws = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")

    def call():
        ops.gpu_attn_chunk_q8_layer(c.desc, c.pages, c.kv, out, q, tok, start, 200, 200, 512, 0, 0, ws, n)

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for new, st in (([200, 0, 0], [0, 0, 0]), ([1, 130, 69], [400, 200, 0]), ([3, 3, 4], [509, 100, 0])):
        tok.copy_(_i32(_starts(new)))
        start.copy_(_i32(st))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        _check_chunk(c, q, out, new, st, 0, 0, "replay")


def test_two_streams_at_once(ops):
    """Calls that overlap on the GPU, each with a workspace of its own, give what they give alone."""
    H, kvH, n = 8, 2, 3000
    c = R.Cache(ops, BF16, 8, H, kvH, n, "paged", 64)
    c.fill([n - 100 * b for b in range(8)])
    lens = _i32([n - 100 * b for b in range(8)])
    qd, qc = _randn((8, H, D), BF16, 3), _randn((8 * 40, H, D), BF16, 4)
    tok, start = _i32(np.arange(9) * 40), lens - 40
    n_d = ops.gpu_attn_decode_q8_workspace_bytes(c.desc, n)
    n_c = ops.gpu_attn_chunk_q8_workspace_bytes(c.desc, 320, 40, n)
    streams = [torch.cuda.Stream() for _ in range(4)]
    ws = [torch.empty(max(n_d, n_c), dtype=torch.uint8, device="cuda") for _ in streams]
    outs = [torch.zeros_like(qc if i % 2 else qd) for i in range(4)]

    def call(i):
        if i % 2:
            ops.gpu_attn_chunk_q8_layer(c.desc, c.pages, c.kv, outs[i], qc, tok, start, 320, 40, n, 0, 0, ws[i], n_c)
        else:
            ops.gpu_attn_decode_q8_layer(c.desc, c.pages, c.kv, outs[i], qd, lens, n, 0, 0, ws[i], n_d)

    want = []
    for i in range(2):
        call(i)
        torch.cuda.synchronize()
        want.append(outs[i].clone())
        outs[i].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                call(i)
    torch.cuda.synchronize()
    for i in range(4):
        assert torch.equal(outs[i], want[i % 2])


# ------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("dt,neox,window,sink", [(BF16, True, 0, 0), (FP16, False, 96, 4)])
def test_serving_run(ops, dt, neox, window, sink):
    """Prompts enter together, are prefilled in two ragged chunks, then decode step by step; on a stream of its own and
    with no wait in between.  Every step is held to 64 bits over the cache that the writer left, and the cache to a
    plain quantiser."""
    H, kvH, B, max_pos = 10, 2, 4, 512
    prompts = [200, 33, 1, 64]
    c = R.Cache(ops, dt, B, H, kvH, max_pos, "paged", 64, neox, seed=8)
    tab = R.rope_table(max_pos)
    tab_d = torch.from_numpy(tab).cuda()
    steps = [[min(p, 100) for p in prompts], [max(0, p - 100) for p in prompts]] + [[1] * B] * 5
    n_dec = ops.gpu_attn_decode_q8_workspace_bytes(c.desc, max_pos)
    n_chk = ops.gpu_attn_chunk_q8_workspace_bytes(c.desc, 400, 100, max_pos)
    ws = torch.empty(max(16, n_dec, n_chk), dtype=torch.uint8, device="cuda")
    side, done, inputs = torch.cuda.Stream(), [0] * B, []
    for i, new in enumerate(steps):
        total = sum(new)
        inputs.append((new, list(done), [_randn((total, h, D), dt, 10 * i + h) for h in (H, kvH, kvH + 100)], _i32(_starts(new)), _i32(done)))
        done = [a + n for a, n in zip(done, new)]
    torch.cuda.synchronize()
    results = []
    with torch.cuda.stream(side):
        for new, start, (q, k, v), tok_d, start_d in inputs:
            total = sum(new)
            v = v[:, :kvH].contiguous()
            qr, out = torch.empty_like(q), torch.full_like(q, 7.0)
            ops.gpu_rope_kv_append_q8_layer(c.desc, c.pages, c.kv, qr, q, k, v, tab_d, tok_d, start_d, total)
            if max(new) == 1 and min(new) == 1:
                ops.gpu_attn_decode_q8_layer(c.desc, c.pages, c.kv, out, qr, start_d + 1, max_pos, window, sink, ws, n_dec)
            else:
                ops.gpu_attn_chunk_q8_layer(c.desc, c.pages, c.kv, out, qr, tok_d, start_d, total, 100, max_pos, window, sink, ws, n_chk)
            results.append((new, start, k, v, qr, out))
    side.synchronize()
    for new, start, k, v, qr, out in results:
        tok = _starts(new)
        for b in range(B):
            if new[b]:
                pos = np.arange(start[b], start[b] + new[b])
                got = c.rows(b, pos)
                rows = slice(tok[b], tok[b + 1])
                for (codes, exps), (gc, gx) in zip((R.quantise(R.rotate_f32(_np32(k[rows]), tab[pos], neox)), R.quantise(_np32(v[rows]))),
                                                   (got[:2], got[2:])):
                    assert np.array_equal(gc.cpu().numpy(), codes) and np.array_equal(gx.cpu().numpy(), exps)
        _check_chunk(c, qr, out, new, start, window, sink, "step")
