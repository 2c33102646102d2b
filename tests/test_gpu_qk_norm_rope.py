"""GPU parity of the fused norm + rotation + cache write (starkv_norm_rope) against the
formula in float64.

Tolerance, per element: half a step of the type (eps / 2 |y|), plus 2^-20 of the row's
largest normed value: f32 carries the mean of at most 128 squares, the root, two products
and a sum (a few 2^-24 each). A table or weight of 16 bits is an input and adds nothing.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda", 0)


def rotary_table(rows, rot, dtype, dev):
    inv = 1.0 / (10000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot))
    a = torch.arange(rows, dtype=torch.float64, device=dev)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).to(dtype)


def formula(x, w, cs, pos, eps):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    rot = cs.shape[1]
    c, s = cs.double()[pos.long()][:, None].chunk(2, -1)
    a, b, rest = y[..., :rot // 2], y[..., rot // 2:rot], y[..., rot:]
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1), y.abs().amax(-1, keepdim=True)


def close(got, want):
    ref, size = want
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + 2.0 ** -20 * size
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25          # half the smallest step
    assert ((got.double() - ref).abs() <= tol).all()


def inputs(n, H, Hkv, D, dtype, seed=0):
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(seed)
    qkv = (torch.randn(n, H + 2 * Hkv, D, generator=g, device=dev) * 2).to(dtype)
    return qkv, (1 + 0.2 * torch.randn(D, generator=g, device=dev)), torch.randint(0, 500, (n,), generator=g, device=dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 64), (128, 64), (128, 48), (64, 16)])
@pytest.mark.parametrize("norm", [True, False])
def test_write(dtype, D, rot, norm):
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope_write
    n, H, Hkv, bs = 37, 6, 2, 16
    qkv, w, pos = inputs(n, H, Hkv, D, dtype, seed=rot)
    dev = qkv.device
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    qw, kw = (w.to(dtype), (w + 0.1).to(dtype)) if norm else (None, None)
    for table_dtype in (torch.float32, torch.bfloat16):
        cs = rotary_table(500, rot, table_dtype, dev)
        kc = torch.full((6, Hkv, bs, D), 5.0, dtype=dtype, device=dev).transpose(1, 2)
        vc = torch.full((6, bs, Hkv, D), 6.0, dtype=dtype, device=dev)
        slots = torch.randperm(6 * bs, device=dev)[:n]
        slots[3], slots[30] = -1, -7                  # padding rows: not written
        k_out = torch.empty(n, Hkv, D, dtype=dtype, device=dev)
        got = qk_norm_rope_write(q, k, v, pos, cs, kc, vc, slots, q_weight=qw, k_weight=kw, eps=1e-5, k_out=k_out)
        close(got, formula(q, qw, cs, pos, 1e-5))
        want = formula(k, kw, cs, pos, 1e-5)
        close(k_out, want)
        live = slots >= 0
        at = slots[live]
        assert torch.equal(kc[at // bs, at % bs], k_out[live])
        assert torch.equal(vc[at // bs, at % bs], v[live])
        untouched = torch.ones(6 * bs, dtype=torch.bool, device=dev)
        untouched[at] = False
        u = untouched.nonzero()[:, 0]
        assert (kc[u // bs, u % bs] == 5).all() and (vc[u // bs, u % bs] == 6).all()


@pytest.mark.parametrize("n,H,Hkv,D", [(1, 32, 8, 128), (1, 1, 1, 64), (3, 5, 5, 64), (1000, 32, 32, 128)])
def test_sizes_and_index_types(n, H, Hkv, D):
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope, qk_norm_rope_write
    qkv, w, pos = inputs(n, H, Hkv, D, torch.bfloat16, seed=n)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    cs = rotary_table(500, D, torch.float16, qkv.device)
    a, b = qk_norm_rope(q, k, pos, cs, q_weight=w, k_weight=w)
    close(a, formula(q, w, cs, pos, 1e-6))
    close(b, formula(k, w, cs, pos, 1e-6))
    blocks = -(-n // 5)
    kc = torch.zeros(blocks, 5, Hkv, D, dtype=torch.bfloat16, device=qkv.device)
    vc = torch.zeros_like(kc)
    slots = torch.arange(n, device=qkv.device, dtype=torch.int32)
    qo = qk_norm_rope_write(q, k, v, pos.int(), cs, kc, vc, slots, q_weight=w, k_weight=w)
    assert torch.equal(qo, a)
    assert torch.equal(kc.view(-1, Hkv, D)[:n], b) and torch.equal(vc.view(-1, Hkv, D)[:n], v)
    only, none = qk_norm_rope(q, None, pos, cs, q_weight=w)
    assert none is None and torch.equal(only, a)


def test_in_place():
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope
    qkv, w, pos = inputs(50, 8, 2, 128, torch.bfloat16)
    cs = rotary_table(500, 128, torch.bfloat16, qkv.device)
    q, k, keep = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:].clone()
    want = qk_norm_rope(q, k, pos, cs, q_weight=w, k_weight=w)
    got = qk_norm_rope(q, k, pos, cs, q_weight=w, k_weight=w, q_out=q, k_out=k)
    assert got[0].data_ptr() == qkv.data_ptr()
    assert torch.equal(qkv[:, :8], want[0]) and torch.equal(qkv[:, 8:10], want[1]) and torch.equal(qkv[:, 10:], keep)


def test_large_and_zero_rows():
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope
    dev = cuda()
    cs = rotary_table(8, 128, torch.float32, dev)
    q = torch.zeros(2, 1, 128, dtype=torch.float16, device=dev)
    q[1] = 60000.0
    w = torch.full((128,), 0.5, device=dev)
    pos = torch.tensor([0, 5], device=dev)
    out, _ = qk_norm_rope(q, None, pos, cs, q_weight=w, eps=1e-6)
    close(out, formula(q, w, cs, pos, 1e-6))
    assert (out[0] == 0).all()


def test_positions_and_slots_outside_are_recorded():
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope, qk_norm_rope_write
    qkv, w, _ = inputs(2, 2, 1, 64, torch.bfloat16)
    dev = qkv.device
    cs = rotary_table(10, 64, torch.bfloat16, dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out, _ = qk_norm_rope(qkv[:, :2], None, torch.tensor([12, -4], device=dev), cs, status=status)
    assert int(status) == 105
    close(out, formula(qkv[:, :2], None, cs, torch.tensor([9, 0], device=dev), 1e-6))
    kc, vc = torch.zeros(2, 2, 4, 1, 64, dtype=torch.bfloat16, device=dev).unbind(0)
    status.zero_()
    qk_norm_rope_write(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], torch.tensor([1, 2], device=dev), cs, kc, vc,
                       torch.tensor([8, 3], device=dev), status=status)
    assert int(status) == 105
    assert torch.equal(vc[0, 3], qkv[1, 3:]) and int((vc != 0).any(-1).sum()) == 1


def test_captured():
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope_write
    qkv, w, pos = inputs(20, 4, 2, 128, torch.bfloat16, seed=9)
    dev = qkv.device
    cs = rotary_table(500, 128, torch.bfloat16, dev)
    kc, vc = torch.zeros(2, 4, 16, 2, 128, dtype=torch.bfloat16, device=dev).unbind(0)
    slots = torch.arange(20, device=dev)
    call = lambda: qk_norm_rope_write(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], pos, cs, kc, vc, slots, q_weight=w,  # noqa
                                      k_weight=w)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    pos.add_(-pos + 7)
    slots.add_(30)
    g.replay()
    torch.cuda.synchronize()
    close(out, formula(qkv[:, :4], w, cs, pos, 1e-6))
    assert torch.equal(vc.view(-1, 2, 128)[30:50], qkv[:, 6:])


def test_write_in_place_and_empty():
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope_write
    qkv, w, pos = inputs(300, 8, 2, 128, torch.bfloat16, seed=12)
    dev = qkv.device
    cs = rotary_table(500, 128, torch.bfloat16, dev)
    kc, vc = torch.zeros(2, 20, 16, 2, 128, dtype=torch.bfloat16, device=dev).unbind(0)
    slots = torch.randperm(320, device=dev)[:300]
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:].clone()
    want = formula(q, w, cs, pos, 1e-6), formula(k, w, cs, pos, 1e-6)
    got = qk_norm_rope_write(q, k, qkv[:, 10:], pos, cs, kc, vc, slots, q_weight=w, k_weight=w, q_out=q, k_out=k)
    assert got.data_ptr() == qkv.data_ptr()
    close(qkv[:, :8], want[0])
    close(qkv[:, 8:10], want[1])
    assert torch.equal(qkv[:, 10:], v)
    assert torch.equal(kc.view(320, 2, 128)[slots], qkv[:, 8:10]) and torch.equal(vc.view(320, 2, 128)[slots], v)
    before = kc.clone()
    none = qk_norm_rope_write(q[:0], k[:0], v[:0], pos[:0], cs, kc, vc, slots[:0])
    assert none.shape == (0, 8, 128) and torch.equal(kc, before)


@pytest.mark.parametrize("H,Hkv,n", [(32, 8, 1000), (7, 3, 2000), (1, 1, 9000), (33, 17, 700), (64, 64, 150)])
@pytest.mark.parametrize("D", [64, 128])
def test_long_batches_of_odd_heads(H, Hkv, n, D):
    """Batches that take the kernel's several-steps form, head counts that leave a step partly
    empty, one norm given and the other not."""
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope_write
    qkv, w, pos = inputs(n, H, Hkv, D, torch.float16, seed=H)
    dev = qkv.device
    cs = rotary_table(500, D, torch.float32, dev)
    kc, vc = torch.zeros(2, -(-n // 16), 16, Hkv, D, dtype=torch.float16, device=dev).unbind(0)
    slots = torch.arange(n, device=dev)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    for qw, kw in ((w, None), (None, w)):
        got = qk_norm_rope_write(q, k, v, pos, cs, kc, vc, slots, q_weight=qw, k_weight=kw)
        close(got, formula(q, qw, cs, pos, 1e-6))
        close(kc.view(-1, Hkv, D)[:n], formula(k, kw, cs, pos, 1e-6))
        assert torch.equal(vc.view(-1, Hkv, D)[:n], v)
