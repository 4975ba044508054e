"""Windowed attention (``gdnx_attn_fwd`` / ``gdnx_attn_bwd``) against the 64-bit oracle.

Tolerances (relative 2-norm).  fp32: a score is off by a few 2^-24 of its size (below 10), sums of n <= 1000
terms by about sqrt(n) 2^-24: 1e-5 holds both with room.  16-bit types round the output once (rms 0.29 of a
spacing: 1.7e-3 in bfloat16, 2.1e-4 in float16) and the weights once before the product with V, whose relative
error is the same and independent: 2.4e-3 and 3e-4 together, twice that is allowed.  The gradients round P and
dS, and read y rounded: four such errors, so again twice the forward's."""
import pytest
import torch

from gdnx_b200 import _lib as L
from gdnx_b200 import ops
from oracle import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TOL = {"f32": 1e-5, "bf16": 5e-3, "f16": 6e-4}
TOL_GRAD = {"f32": 2e-5, "bf16": 1e-2, "f16": 1.2e-3}


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def make(B, Tq, Tk, H, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda T, h: torch.randn(B, T, h, D, generator=g).to(TYPES[dtype]).to(DEV)  # noqa: E731
    return r(Tq, H), r(Tk, Hk), r(Tk, Hk), r(Tq, H)


def check(q, k, v, dy, dtype, **mask):
    """Forward, lse and gradients against the oracle."""
    y, lse = ops.window_attention(q, k, v, return_lse=True, **mask)
    yo, lo = A.window_attention(q, k, v, **mask)
    assert y.dtype == q.dtype and rel(y, yo) < TOL[dtype]
    seen = torch.isfinite(lo)
    assert torch.equal(torch.isfinite(lse).cpu(), seen)
    # the scores' own rounding: products of 16-bit values are exact in fp32
    assert (lse.cpu().double()[seen] - lo[seen]).abs().max().item() < 1e-4 if seen.any() else True
    if dy is None:
        return
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    yt = ops.window_attention_train(q, k, v, **mask)
    assert torch.equal(yt.detach(), y)
    for x, g, go in zip((q, k, v), torch.autograd.grad(yt, (q, k, v), dy), A.window_attention_grads(q, k, v, dy, **mask)):
        assert g.shape == x.shape and g.dtype == x.dtype
        assert torch.isfinite(g).all()
        assert rel(g, go) < TOL_GRAD[dtype] or go.norm() < 1e-12 and g.norm() < 1e-5


SHAPES = [  # B, Tq, Tk, H, Hk, D, window, sinks
    (1, 1, 1, 1, 1, 64, 1, 0),            # one token
    (2, 1, 300, 4, 2, 64, 50, 3),         # one query at the end of a long sequence
    (1, 130, 130, 2, 1, 128, 1, 0),       # a window of one: every query sees itself
    (1, 200, 200, 2, 2, 128, 1, 5),       # and the sinks
    (2, 257, 257, 4, 2, 64, 64, 4),       # one row past a tile
    (1, 384, 384, 6, 3, 128, 100, 0),     # window edges inside tiles
    (1, 500, 500, 2, 1, 96, 129, 130),    # sinks over more than one tile, a head size that is padded
    (1, 300, 300, 5, 1, 80, 1000, 4),     # window beyond the sequence: plain causal
    (2, 100, 421, 4, 4, 32, 333, 17),     # a continued prompt
    (1, 129, 640, 16, 1, 128, 200, 64),   # 16 query heads of one key head
    (1, 640, 640, 2, 1, 8, 200, 1000),    # sinks beyond the sequence; the smallest head
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_and_gradients(shape, dtype):
    B, Tq, Tk, H, Hk, D, window, sinks = shape
    check(*make(B, Tq, Tk, H, Hk, D, dtype, seed=Tk), dtype, window=window, sinks=sinks)


ODD = [  # an odd number of query heads for each key head: two consecutive blocks of queries share their tiles, and the
    # second sees the sinks' tile but not the first of the window's; more items than SMs
    (1, 3000, 3000, 16, 16, 64, 200, 4),
    (3, 1100, 1100, 16, 16, 128, 130, 17),
    (2, 2200, 2500, 15, 5, 96, 700, 130),
    (1, 2600, 2600, 5, 1, 32, 60, 1),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", ODD, ids=str)
def test_blocks_that_share_tiles_with_a_gap(shape, dtype):
    B, Tq, Tk, H, Hk, D, window, sinks = shape
    q, k, v, dy = make(B, Tq, Tk, H, Hk, D, dtype, seed=Tk)
    lengths = torch.arange(Tk, Tk - 70 * B, -70, device=DEV, dtype=torch.int32)
    for _ in range(3):
        check(q, k, v, None, dtype, window=window, sinks=sinks, lengths=lengths)
    check(q, k, v, dy, dtype, window=window, sinks=sinks, lengths=lengths)
    assert ops.device_status() == 0


FEW = [  # few enough blocks that each has a CTA of its own (one tile, an odd number of them, sinks apart from the window;
    # one block too many for that), and a last round that is nearly empty
    (1, 128, 128, 2, 2, 128, 50, 0),
    (1, 300, 300, 1, 1, 64, 300, 0),
    (1, 257, 900, 4, 2, 96, 130, 7),
    (2, 640, 640, 8, 2, 128, 4000, 4),
    (1, 128, 700, 149, 1, 64, 200, 3),
    (1, 1280, 1280, 30, 15, 128, 60, 4),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", FEW, ids=str)
def test_blocks_whose_keys_are_split(shape, dtype):
    B, Tq, Tk, H, Hk, D, window, sinks = shape
    q, k, v, dy = make(B, Tq, Tk, H, Hk, D, dtype, seed=Tq)
    lengths = torch.arange(Tk, Tk - 70 * B, -70, device=DEV, dtype=torch.int32)
    check(q, k, v, dy, dtype, window=window, sinks=sinks, lengths=lengths)
    empty = torch.zeros(B, device=DEV, dtype=torch.int32)
    assert not ops.window_attention(q, k, v, window=window, sinks=sinks, lengths=empty).any()
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Tq,Tk,D", [(260, 260, 128), (70, 260, 64)])
def test_padding_holds_nan_and_reaches_nothing(Tq, Tk, D, dtype):
    """Lengths 0, 1, inside a tile, a tile's edge and full; what lies beyond them is NaN."""
    n = [0, 1, 128, 201, Tk, 64]
    q, k, v, dy = make(len(n), Tq, Tk, 4, 2, D, dtype, seed=5)
    for b, m in enumerate(n):
        k[b, m:] = float("nan")
        v[b, m:] = float("inf")
        q[b, max(0, m - (Tk - Tq)):] = float("nan")
        dy[b, max(0, m - (Tk - Tq)):] = float("nan")
    lengths = torch.tensor(n, dtype=torch.int32, device=DEV)
    check(q, k, v, dy, dtype, window=90, sinks=4, lengths=lengths)
    y = ops.window_attention(q, k, v, window=90, sinks=4, lengths=lengths)
    for b, m in enumerate(n):
        assert (y[b, max(0, m - (Tk - Tq)):] == 0).all()


def test_lengths_out_of_range_are_clamped():
    q, k, v, _ = make(2, 40, 40, 2, 2, 64, "bf16")
    y = ops.window_attention(q, k, v, lengths=torch.tensor([-3, 99], dtype=torch.int32, device=DEV))
    assert (y[0] == 0).all() and torch.equal(y[1], ops.window_attention(q, k, v)[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_orders(dtype):
    """Heads before tokens, a slice of a wider projection, an odd row stride, a shared batch."""
    q, k, v, dy = make(2, 150, 150, 4, 2, 64, dtype, seed=3)
    mask = dict(window=70, sinks=2)
    want = ops.window_attention(q, k, v, **mask)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(ops.window_attention(*heads_first, **mask), want)
    wide = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1)
    a = wide[..., :256].unflatten(2, (4, 64)), wide[..., 256:384].unflatten(2, (2, 64)), wide[..., 384:].unflatten(2, (2, 64))
    assert torch.equal(ops.window_attention(*a, **mask), want)
    check(*a, dy.transpose(1, 2).contiguous().transpose(1, 2), dtype, **mask)
    odd = torch.empty(2, 150, 4, 67, dtype=q.dtype, device=DEV)[..., 1:65]
    odd.copy_(q)
    check(odd, k, v, dy, dtype, **mask)
    check(q, k[:1].expand(2, -1, -1, -1), v[:, :, :1].expand(-1, -1, 2, -1), dy, dtype, **mask)


def test_gradients_of_broadcast_inputs_are_summed():
    q, k, v, dy = make(3, 90, 90, 4, 4, 64, "f32", seed=8)
    k1, v1 = k[:1].detach().requires_grad_(), v[:, :, :1].detach().requires_grad_()
    y = ops.window_attention_train(q, k1.expand(3, -1, -1, -1), v1.expand(-1, -1, 4, -1), window=30, sinks=2)
    dk, dv = torch.autograd.grad(y, (k1, v1), dy)
    _, gk, gv = A.window_attention_grads(q, k1.expand(3, -1, -1, -1), v1.expand(-1, -1, 4, -1), dy, window=30, sinks=2)
    assert rel(dk, gk.sum(0, keepdim=True)) < 2e-5 and rel(dv, gv.sum(2, keepdim=True)) < 2e-5


def test_gradient_of_a_sum_is_taken():
    """A cotangent with stride 0 everywhere."""
    q, k, v, _ = make(1, 50, 50, 2, 2, 64, "f32", seed=9)
    v.requires_grad_()
    ops.window_attention_train(q, k, v, window=20).sum().backward()
    _, _, gv = A.window_attention_grads(q, k, v, torch.ones_like(q), window=20)
    assert rel(v.grad, gv) < 2e-5


def test_gradients_against_differences():
    """fp32: the loss's change over +-h along random directions against the gradient's share in them.  With h = 1e-2
    the third-order term is below h^2 = 1e-4 of the slope, the rounding of a loss of about 100 below 1e-5 / h."""
    q, k, v, dy = make(1, 70, 70, 2, 1, 32, "f32", seed=11)
    mask = dict(window=33, sinks=2)
    xs = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.window_attention_train(*xs, **mask), xs, dy)
    loss = lambda t: (ops.window_attention(*t, **mask).double() * dy.double()).sum().item()  # noqa: E731
    h = 1e-2
    for i, g in enumerate(grads):
        e = torch.randn(g.shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        e = e / e.norm()
        up, down = [q, k, v], [q, k, v]
        up[i], down[i] = up[i] + h * e, down[i] - h * e
        slope = (loss(up) - loss(down)) / (2 * h)
        assert abs(slope - (g.double() * e.double()).sum().item()) < 2e-3 * g.double().norm().item()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores_and_scale(dtype):
    """Scores of hundreds: the running maximum has to carry them."""
    q, k, v, dy = make(1, 200, 200, 2, 1, 64, dtype, seed=12)
    y = ops.window_attention(q * 8, k * 8, v, window=150, scale=0.5)
    yo, _ = A.window_attention(q * 8, k * 8, v, window=150, scale=0.5)
    # a score of 500 carries 500 2^-24 = 3e-5 into its weight
    assert rel(y, yo) < max(TOL[dtype], 1e-4)


def test_same_inputs_give_the_same_bits():
    q, k, v, dy = make(2, 700, 700, 8, 2, 128, "bf16", seed=13)
    runs = []
    for _ in range(3):
        xs = [t.detach().requires_grad_() for t in (q, k, v)]
        y = ops.window_attention_train(*xs, window=200, sinks=4)
        runs.append([y.detach(), *torch.autograd.grad(y, xs, dy)])
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)


def test_gradient_of_a_gradient_is_refused():
    q, k, v, dy = make(1, 20, 20, 2, 2, 64, "f32")
    q.requires_grad_()
    y = ops.window_attention_train(q, k, v)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y, q, dy, create_graph=True)


def test_out_dtype_and_out():
    q, k, v, _ = make(2, 150, 150, 4, 2, 128, "bf16", seed=14)
    yo, _ = A.window_attention(q, k, v, window=60)
    y32 = ops.window_attention(q, k, v, window=60, out_dtype=torch.float32)
    assert y32.dtype == torch.float32 and rel(y32, yo) < TOL["bf16"]
    buf = torch.full((2, 150, 4, 160), 7.0, dtype=torch.bfloat16, device=DEV)
    out = buf[..., 16:144]
    assert ops.window_attention(q, k, v, window=60, out=out) is out
    assert rel(out, yo) < TOL["bf16"] and (buf[..., :16] == 7).all() and (buf[..., 144:] == 7).all()
    odd = torch.full((2, 150, 4, 131), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.window_attention(q, k, v, window=60, out=odd[..., 1:129])
    assert rel(odd[..., 1:129], yo) < TOL["bf16"] and (odd[..., :1] == 7).all() and (odd[..., 129:] == 7).all()


def test_on_another_stream():
    q, k, v, _ = make(1, 300, 300, 4, 2, 64, "bf16", seed=15)
    want = ops.window_attention(q, k, v, window=100)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.window_attention(q * 1, k, v, window=100)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype,B,T", [("bf16", 1, 700), ("bf16", 4, 1500), ("f32", 2, 300)])
def test_in_a_graph(dtype, B, T):
    """A captured step (kernels that start beside their predecessors among them) replayed on new inputs."""
    q, k, v, dy = make(B, T, T, 6, 3, 128, dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]

    def step():
        y = ops.window_attention_train(*leaves, window=100, sinks=4)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        with torch.no_grad():
            for t, new in zip((*leaves, dy), make(B, T, T, 6, 3, 128, dtype, seed=seed)):
                t.copy_(new)
        graph.replay()
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    assert ops.device_status() == 0


def test_empty_sizes():
    q, k, v, _ = make(2, 3, 5, 2, 1, 64, "bf16")
    assert ops.window_attention(q[:0], k[:0], v[:0]).shape == (0, 3, 2, 64)
    assert ops.window_attention(q[:, :0], k[:, :0], v[:, :0]).shape == (2, 0, 2, 64)
    xs = [t.detach().requires_grad_() for t in (q[:, :0], k, v)]
    y = ops.window_attention_train(*xs)
    dq, dk, dv = torch.autograd.grad(y, xs, torch.zeros_like(y))
    assert dq.shape == (2, 0, 2, 64) and (dk == 0).all() and (dv == 0).all()


def test_refusals():
    q, k, v, _ = make(2, 8, 8, 4, 2, 64, "bf16")
    bad = [dict(window=0), dict(sinks=-1), dict(lengths=torch.zeros(3, dtype=torch.int32, device=DEV)),
           dict(lengths=torch.zeros(2, dtype=torch.int64, device=DEV)), dict(lengths=torch.zeros(2, dtype=torch.int32)),
           dict(out=torch.empty(2, 8, 4, 32, dtype=q.dtype, device=DEV))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.window_attention(q, k, v, **kw)
    for a in ((q, k[:, :4], v[:, :4]), (q, k[:1], v[:1]), (q[:, :, :3], k, v), (q, k, v[:, :4]), (q[0], k, v),
              (q, k[..., :32], v[..., :32]), (q.transpose(2, 3), k, v)):
        with pytest.raises(ValueError):
            ops.window_attention(*a)
    for a in ((q.float(), k, v), (q, k, v.half()), (q.double(), k.double(), v.double())):
        with pytest.raises(TypeError):
            ops.window_attention(*a)
    with pytest.raises(L.GdnxError) as e:
        ops.window_attention(q, k, v, scale=-1.0)
    assert e.value.status == L.GDNX_EINVAL
    wide = torch.zeros(1, 4, 1, 136, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(L.GdnxError) as e:
        ops.window_attention(wide, wide, wide)
    assert e.value.status == L.GDNX_EUNSUPPORTED


def test_offsets_beyond_32_bits():
    """Batch rows more than 2^31 elements apart, for the inputs and the output."""
    far = (1 << 31) + 64
    n = 40 * 2 * 64
    bufs = [torch.empty(far + n, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    parts = [make(2, 40, 40, 2, 2, 64, "bf16", seed=20)[i] for i in range(3)]
    q, out = (b.as_strided((2, 40, 2, 64), (far, 128, 64, 1)) for b in bufs)
    q.copy_(parts[0])
    ops.window_attention(q, parts[1], parts[2], window=9, sinks=1, out=out)
    assert torch.equal(out, ops.window_attention(*parts, window=9, sinks=1))
    f = [t.float() for t in parts]
    del bufs, q, out
    buf = torch.empty(far + n, dtype=torch.float32, device=DEV)
    q = buf.as_strided((2, 40, 2, 64), (far, 128, 64, 1))
    q.copy_(f[0])
    assert torch.equal(ops.window_attention(q, f[1], f[2], window=9), ops.window_attention(*f, window=9))


def _same_where_finite(got, want, tol):
    """NaN where the other is, close elsewhere."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert rel(got.nan_to_num(0), want.nan_to_num(0)) < tol


BAD_KEYS = {  # a key's first value where the queries' first value is positive, and what else its row holds
    "nan": float("nan"), "score inf": float("inf"), "score -inf": -float("inf")}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,H", [(1, 150, 2), (1, 150, 1), (5, 1000, 4)])  # keys of a block split over the stages, and not
@pytest.mark.parametrize("what", BAD_KEYS)
def test_scores_that_are_not_finite_show_in_their_rows(what, B, T, H, dtype):
    """A row that sees a score of NaN or +inf is NaN whatever the key's place in its tile, one that sees -inf only too;
    other rows do not notice.  The same for the log of the sum."""
    for j in (0, 1, 6, 7, 45, 134) if B == 1 else (1, 6, 134):
        q, k, v, _ = make(B, T, T, H, H, 64, dtype, seed=j)
        q[..., 0] = 1.0
        k[:, j] = 0.0
        k[:, j, :, 0] = BAD_KEYS[what]
        y, lse = ops.window_attention(q, k, v, window=40, return_lse=True)
        yo, lo = A.window_attention(q, k, v, window=40)
        assert yo.isnan().any() or what == "score -inf" and j > 0
        _same_where_finite(y, yo, TOL[dtype])
        _same_where_finite(lse, lo, 1e-5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_that_overflow_show_in_their_rows(dtype):
    """Finite inputs whose product leaves fp32's range, at every place of a run of 16 keys."""
    for j in range(16):
        q, k, v, _ = make(1, 60, 60, 2, 2, 64, dtype, seed=j)
        q[..., 0] = 1e20
        k[:, :, :, 0] = 0.0
        k[:, j, :, 0] = 1e20
        y, lse = ops.window_attention(q, k, v, return_lse=True)
        assert y[:, j:].isnan().all() and lse[..., j:].isnan().all()
        assert y[:, :j].isfinite().all() and lse[..., :j].isfinite().all()
        y = ops.window_attention(q, -k, v)
        assert y[:, j + 1:].isfinite().all() and y[:, :j].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", [1, 5, 6, 7, 48, 130])
def test_a_query_that_is_not_finite_shows_in_its_gradients(i, dtype):
    """NaN in a query: in its own dq, and in dk and dv of every key that it sees, whatever its place in the tile; nothing
    of other heads notices."""
    q, k, v, dy = make(1, 200, 200, 4, 2, 64, dtype, seed=i)
    q[:, i, 1] = float("nan")
    xs = [t.detach().requires_grad_() for t in (q, k, v)]
    y = ops.window_attention_train(*xs, window=70, sinks=2)
    dq, dk, dv = torch.autograd.grad(y, xs, dy)
    seen = A.visible(200, 200, 70, 2)[i].to(DEV)
    assert y[:, i, 1].isnan().all() and dq[:, i, 1].isnan().all()
    assert dk[:, seen, 0].isnan().all() and dv[:, seen, 0].isnan().all()
    assert dq[:, :, [0, 2, 3]].isfinite().all() and dk[:, :, 1].isfinite().all() and dv[:, :, 1].isfinite().all()


def _run(code):
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]


def test_the_first_call_may_be_captured():
    """A process whose first attention calls happen while a graph is captured."""
    _run("""
import torch
from gdnx_b200 import ops
q, k, v = (torch.randn(1, 300, 2, 64, device="cuda").to(torch.bfloat16).requires_grad_() for _ in range(3))
dy = torch.randn_like(q)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ops.window_attention_train(q, k, v, window=50)
    grads = torch.autograd.grad(y, (q, k, v), dy)
graph.replay()
want = ops.window_attention_train(q, k, v, window=50)
assert torch.equal(y, want)
assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, (q, k, v), dy)))
assert ops.device_status() == 0
""")


def test_the_error_word_is_one_word_and_can_be_cleared():
    """Threads that ask for it at once get the same word; what a kernel leaves there is read, told and cleared."""
    import threading
    ops.clear_device_status()
    ops._ERRORS.clear()
    words, gate, zeros = [], threading.Barrier(4), torch.zeros

    def meet(*a, **kw):  # were a word made by the asking thread, all four would make theirs here
        gate.wait(timeout=60)
        return zeros(*a, **kw)

    def ask():
        gate.wait(timeout=60)
        words.append(ops._error_word(0))

    torch.zeros = meet
    try:
        threads = [threading.Thread(target=ask) for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        torch.zeros = zeros
    assert len(words) == 4 and len(set(words)) == 1

    class Word:
        __cuda_array_interface__ = dict(shape=(1,), typestr="<i4", data=(words[0], False), version=2)

    word = torch.as_tensor(Word(), device=DEV)
    assert word.data_ptr() == words[0]
    word.fill_(L.GDNX_ETIMEOUT)
    assert ops.device_status() == L.GDNX_ETIMEOUT
    with pytest.raises(RuntimeError, match="ETIMEOUT"):
        ops.check_device_status()
    ops.clear_device_status()
    assert ops.device_status() == 0 and int(word) == 0
    ops.check_device_status()


def _forward_args(q, k, v, lengths):
    a, index = ops._attn_args(q, k, v, 16, 2, None, lengths)
    y, lse = torch.empty_like(q), torch.empty(q.shape[0], q.shape[2], q.shape[1], device=DEV)
    a.y, a.y_dtype, a.lse = y.data_ptr(), ops._DT[y.dtype], lse.data_ptr()
    a.y_sb, a.y_st, a.y_sh, _ = y.stride()
    return a, (y, lse)


@pytest.mark.parametrize("dtype", TYPES)
def test_c_entries_refuse_pointers_between_elements(dtype):
    """Refused on the host, before any launch.  (Every address asked for lies inside its tensor.)"""
    import ctypes as C
    lib = L.load()
    lengths = torch.full((2,), 24, dtype=torch.int32, device=DEV)
    q, k, v, dy = make(2, 32, 32, 4, 2, 64, dtype)

    def moved(s, field, by, call, status=L.GDNX_EINVAL):
        at = s
        *path, last = field.split(".")
        for name in path:
            at = getattr(at, name)
        was = getattr(at, last)
        setattr(at, last, was + by)
        assert call() == status, field
        setattr(at, last, was)

    a, keep = _forward_args(q, k, v, lengths)
    forward = lambda: lib.gdnx_attn_fwd(C.byref(a), None)  # noqa: E731
    for field in ("q.ptr", "k.ptr", "v.ptr", "y", "lse", "lengths", "error"):
        moved(a, field, 1, forward)
    g = L.AttnBwdArgs(a, ops._heads_view(dy))
    grads = [torch.empty_like(t) for t in (q, k, v)]
    g.dq, g.dk, g.dv = (t.data_ptr() for t in grads)
    ws = torch.empty(lib.gdnx_attn_bwd_workspace_bytes(C.byref(g)) + 16, dtype=torch.uint8, device=DEV)
    g.workspace, g.workspace_bytes = ws.data_ptr(), ws.numel() - 16
    backward = lambda: lib.gdnx_attn_bwd(C.byref(g), None)  # noqa: E731
    for field in ("fwd.q.ptr", "fwd.lse", "dy.ptr", "dq", "dk", "dv"):
        moved(g, field, 1, backward)
    moved(g, "workspace", 1, backward, L.GDNX_EWORKSPACE)

    c = ops.PagedCache.zeros(1, 200, 2, 16, 64, slots=2, width=100, dtype=TYPES[dtype], device=DEV)
    rows = torch.arange(2, dtype=torch.int32, device=DEV)
    s, _ = ops._cache_struct(c)
    y = torch.empty_like(q[:, 0])
    d = L.PagedDecodeArgs(s, 2, 4, 0, 1 << 40, 0, 0, 0.125, ops._heads_view(q[:, :1]), rows.data_ptr(), y.data_ptr(),
                          ops._DT[y.dtype], 256, 64, ops._error_word(0))
    room = torch.empty(lib.gdnx_paged_decode_workspace_bytes(C.byref(d)) + 16, dtype=torch.uint8, device=DEV)
    assert room.numel() > 16
    d.workspace, d.workspace_bytes = room.data_ptr(), room.numel() - 16
    decode = lambda: lib.gdnx_paged_decode(C.byref(d), None)  # noqa: E731
    for field in ("q.ptr", "y", "rows", "error", "cache.table", "cache.lengths", "cache.refs", "cache.status"):
        moved(d, field, 1, decode)
    moved(d, "cache.kv", 8, decode)
    moved(d, "workspace", 8, decode, L.GDNX_EWORKSPACE)
    kv = ops._heads_view(k)
    for by in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        at = L.View.from_buffer_copy(kv)
        at.ptr += by[0]
        assert lib.gdnx_cache_write(C.byref(s), 0, 2, 32, C.byref(at), C.byref(kv), rows.data_ptr() + by[1],
                                    lengths.data_ptr() + by[2], None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_truncate(C.byref(s), 1, rows.data_ptr() + 2, rows.data_ptr(), None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_extend(C.byref(s), 1, rows.data_ptr(), rows.data_ptr(), room.data_ptr() + 1, 1 << 40,
                                 None) == L.GDNX_EWORKSPACE
    assert lib.gdnx_cache_compact(C.byref(s), room.data_ptr() + 2, 1 << 40, None) == L.GDNX_EWORKSPACE
    torch.cuda.synchronize()
    ops.cache_check(c)


@pytest.mark.parametrize("T,H,Hk,window,sinks", [(1500, 64, 16, 60, 900), (1100, 16, 16, 40, 1100), (900, 12, 4, 128, 300)])
def test_gradients_where_many_keys_are_sinks(T, H, Hk, window, sinks):
    """Key tiles that every later query sees, cut into parts of more than a tile's own length, into such parts, and whole."""
    check(*make(1, T, T, H, Hk, 64, "bf16", seed=T), "bf16", window=window, sinks=sinks)
