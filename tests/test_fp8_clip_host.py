"""What autolabel_amd.fp8 and autolabel_amd.clip refuse, and what their C entry points refuse, without a GPU: every case here is turned away
on the host before anything is launched."""
import ctypes as C
import math

import pytest
import torch

from autolabel_amd import clip, fp8, hip


def blocks(rows, cols, fmt='e4m3'):
    nb = (cols + 127) // 128
    return fp8.Fp8Blocks(torch.zeros(rows, nb * 128).to(fp8.FORMATS[fmt][1]), torch.full((rows, (nb + 3) // 4 * 4), 127, dtype=torch.uint8), cols, fmt)


def test_blocks_are_checked():
    good = blocks(8, 200)
    good._check('x')
    for bad in (dict(fmt='e3m4'), dict(cols=0), dict(cols=257), dict(q=good.q.float()), dict(q=good.q[:, :130]), dict(q=good.q[0]), dict(scale=good.scale[:7]),
                dict(scale=good.scale[:, :1]), dict(scale=good.scale.int()), dict(fmt='e5m2')):
        with pytest.raises(ValueError):
            fp8.Fp8Blocks(**{**dict(q=good.q, scale=good.scale, cols=200, fmt='e4m3'), **bad})._check('x')
    assert good.rows == 8 and good.dequantize().shape == (8, 200)


def test_dequantize_values():
    b = blocks(2, 130)
    b.q[0, 0], b.q[1, 129] = 1.5, -448.0
    b.scale[0, 0], b.scale[1, 1] = 130, 1
    v = b.dequantize()
    assert v[0, 0] == 12.0 and v[1, 129] == -448.0 * 2.0 ** -126 and v.abs().sum() == v[0, 0] - v[1, 129]


@pytest.mark.parametrize('call, match', [
    (lambda: fp8.quantize(torch.zeros(3, 4)), 'no CPU path'),
    (lambda: fp8.quantize(torch.zeros(3, 4), fmt='e3m4'), 'unknown 8-bit format'),
    (lambda: fp8.quantize(torch.zeros(3, 4, dtype=torch.float64)), 'fp16, bf16 or fp32'),
    (lambda: fp8.quantize(torch.zeros(3, 4, dtype=torch.int8)), 'fp16, bf16 or fp32'),
    (lambda: fp8.quantize(torch.zeros(())), 'at least one column'),
    (lambda: fp8.quantize(torch.zeros(3, 0)), 'at least one column'),
    (lambda: fp8.quantize(torch.zeros(0, 4), transpose=True), 'empty x'),
    (lambda: fp8.matmul(blocks(2, 128), blocks(2, 129)), 'contract over'),
    (lambda: fp8.matmul(blocks(2, 128), blocks(0, 128)), 'no rows'),
    (lambda: fp8.matmul(blocks(2, 128), blocks(2, 128), torch.float64), 'results are'),
    (lambda: fp8.matmul(blocks(2, 128), blocks(2, 128)), 'no CPU path'),
    (lambda: fp8.linear(torch.zeros(2, 128), torch.zeros(2, 128)), 'must be Fp8Blocks'),
    (lambda: fp8.linear(torch.zeros(2, 127), blocks(2, 128)), 'columns'),
    (lambda: fp8.linear(torch.zeros(2, 128), blocks(2, 128), out_dtype=torch.int32), 'results are'),
    (lambda: fp8.linear(torch.zeros(2, 128), blocks(2, 128), fmt='x'), 'unknown 8-bit format'),
    (lambda: fp8.linear_backward(torch.zeros(3, 2), torch.zeros(4, 128), blocks(128, 2)), 'rows'),
    (lambda: fp8.linear_backward(torch.zeros(4, 2), torch.zeros(4, 128), blocks(2, 128)), 'weight_t is'),
    (lambda: fp8.linear_backward(torch.zeros(4, 2), torch.zeros(4, 128), None), 'weight_t must be'),
    (lambda: fp8.linear_backward(torch.zeros(4, 2), torch.zeros(4, 128), blocks(128, 2), grad_fmt='x'), 'unknown 8-bit format'),
    (lambda: fp8.Linear(4, 4, grad_fmt='x'), 'unknown 8-bit format'),
    (lambda: clip.clip_grad_norm_([], 1.0), 'empty list'),
    (lambda: clip.clip_grad_norm_([torch.zeros(3)], 1.0), 'no CPU path'),
    (lambda: clip.clip_grad_norm_([torch.zeros(3)], -1.0), 'max_norm'),
    (lambda: clip.clip_grad_norm_([torch.zeros(3)], math.nan), 'max_norm'),
    (lambda: clip.clip_grad_norm_([torch.zeros(3, dtype=torch.float64)], 1.0), 'dense fp16'),
    (lambda: clip.clip_grad_norm_([torch.zeros(3).to_sparse()], 1.0), 'dense fp16'),
    (lambda: clip.clip_grad_norm_([None], 1.0), 'dense fp16'),
    (lambda: clip.clip_grad_norm_([torch.zeros(4, 4)[:, :2]], 1.0), 'one run of memory'),
    (lambda: clip.clip_grad_norm_([torch.zeros(1).expand(5)], 1.0), 'one run of memory'),
    (lambda: clip.clip_grad_norm_([torch.zeros(3)], 1.0, out=[]), 'outputs'),
    (lambda: clip.clip_grad_norm_([torch.zeros(3)], 1.0, out=[torch.zeros(4)]), 'output 0'),
    (lambda: clip.clip_grad_norm_([torch.zeros(3)], 1.0, loss_scale=2.0), 'loss_scale'),
    (lambda: clip.clip_grad_norm_([torch.zeros(3)], 1.0, found_inf=torch.zeros(1)), 'found_inf'),
    (lambda: clip.grad_norm([]), 'empty list'),
])
def test_python_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_dense_layouts():
    t = torch.zeros(2, 3, 4, 5)
    for good in (t, t.permute(3, 1, 0, 2), t.to(memory_format=torch.channels_last), t[:1], torch.zeros(()), torch.zeros(0, 3), t[:, :, :, :1][0, 0, :1]):
        assert clip._dense(good)
    for bad in (t[:, :2], t[..., ::2], torch.zeros(1, 4).expand(3, 4)):
        assert not clip._dense(bad)


# the C entry points: pointers that are never followed (every call fails on the host)
A = 1 << 20        # aligned to everything
ARGS = {
    'aln_fp8_quantize': dict(x=A, x_type=0, ldx=256, M=4, K=200, fmt=0, q=A, ldq=256, scale=A, lds=4, stream=None),
    'aln_fp8_quantize_t': dict(x=A, x_type=0, ldx=256, M=4, K=200, fmt=0, q=A, ldq=128, scale=A, lds=4, stream=None),
    'aln_fp8_nt': dict(a=A, lda=256, sa=A, ldsa=4, fmt_a=0, b=A, ldb=256, sb=A, ldsb=4, fmt_b=0, M=4, N=8, K=200, y=A, ldy=8, y_type=0, relu=0, ws=None, ws_bytes=0, stream=None),
}


@pytest.mark.parametrize('name, bad, match', [
    ('aln_fp8_quantize', dict(x=None), 'NULL'), ('aln_fp8_quantize', dict(x=A + 1), 'aligned to its type'), ('aln_fp8_quantize', dict(x_type=3), 'unknown type'),
    ('aln_fp8_quantize', dict(fmt=2), 'format'), ('aln_fp8_quantize', dict(M=-1), 'values'), ('aln_fp8_quantize', dict(M=1 << 31), 'values'),
    ('aln_fp8_quantize', dict(K=0), 'values'), ('aln_fp8_quantize', dict(ldx=-1), 'pitch'), ('aln_fp8_quantize', dict(q=None), '8-bit blocks'),
    ('aln_fp8_quantize', dict(q=A + 8), '8-bit blocks'), ('aln_fp8_quantize', dict(ldq=240), '8-bit blocks'), ('aln_fp8_quantize', dict(ldq=264), '8-bit blocks'),
    ('aln_fp8_quantize', dict(scale=None), '8-bit blocks'), ('aln_fp8_quantize', dict(scale=A + 2), '8-bit blocks'), ('aln_fp8_quantize', dict(lds=2), '8-bit blocks'),
    ('aln_fp8_quantize_t', dict(M=129), '8-bit blocks'), ('aln_fp8_quantize_t', dict(M=700, ldq=768), '8-bit blocks'),
    ('aln_fp8_nt', dict(fmt_a=7), 'unknown format'), ('aln_fp8_nt', dict(y_type=-1), 'unknown format'), ('aln_fp8_nt', dict(N=0), 'sizes'), ('aln_fp8_nt', dict(K=0), 'sizes'),
    ('aln_fp8_nt', dict(ldy=7), 'sizes'), ('aln_fp8_nt', dict(a=None), '8-bit blocks'), ('aln_fp8_nt', dict(sb=None), '8-bit blocks'), ('aln_fp8_nt', dict(ldb=128), '8-bit blocks'),
    ('aln_fp8_nt', dict(y=None), 'y is NULL'), ('aln_fp8_nt', dict(y=A + 2, y_type=2), 'y is NULL'),
    ('aln_fp8_nt', dict(K=4096, lda=4096, ldb=4096, ldsa=32, ldsb=32), 'workspace'),
])
def test_c_refusals(name, bad, match):
    args = {**ARGS[name], **bad}
    with pytest.raises(RuntimeError, match=match):
        hip.call(name, *args.values())


def grad_clip(grads=(A, A + 4096), numel=(10, 10), types=(2, 2), out=None, max_norm=1.0, apply=1, ws=A, ws_bytes=1 << 14):
    n = len(grads)
    arr = lambda t, v: (t * len(v))(*v) if v is not None else None
    hip.call('aln_grad_clip', n, arr(C.c_void_p, grads), arr(C.c_void_p, out), arr(C.c_int64, numel), arr(C.c_int32, types), max_norm, apply, None, None, None, ws, ws_bytes, None)


@pytest.mark.parametrize('bad, match', [
    (dict(grads=(), numel=(), types=()), 'empty list'), (dict(max_norm=-1.0), 'max_norm'), (dict(max_norm=math.nan), 'max_norm'), (dict(ws=None), 'workspace'),
    (dict(ws_bytes=100), 'workspace'), (dict(types=(2, 3)), 'unknown type'), (dict(numel=(10, -1)), 'elements'), (dict(grads=(A, None)), 'NULL'),
    (dict(grads=(A, A + 4098)), 'not aligned'), (dict(grads=(A, A)), 'share memory'), (dict(grads=(A, A + 36)), 'share memory'),
    (dict(out=(A, A)), 'share memory'), (dict(out=(A + 4096, A)), 'share memory'), (dict(out=(A, None)), 'output 1'), (dict(out=(A + 8192, A + 8200)), 'share memory'),
])
def test_grad_clip_c_refusals(bad, match):
    with pytest.raises(RuntimeError, match=match):
        grad_clip(**bad)


def test_workspace_sizes():
    L = hip.lib()
    assert L.aln_fp8_nt_ws_bytes(0, 5, 5) == 0 and L.aln_fp8_nt_ws_bytes(1 << 20, 512, 512) == 0
    assert L.aln_fp8_nt_ws_bytes(512, 512, 1 << 20) % (512 * 512 * 4) == 0 and L.aln_fp8_nt_ws_bytes(512, 512, 1 << 20) > 0
    assert L.aln_grad_clip_ws_bytes(1) == L.aln_grad_clip_ws_bytes(120) > 0 and L.aln_grad_clip_ws_bytes(121) == 2 * L.aln_grad_clip_ws_bytes(120)


def test_engine_and_trainer_refusals():
    from autolabel_amd.engine import TrainEngine
    from autolabel_amd.trainer import Trainer
    with pytest.raises(ValueError, match='max_grad_norm'):
        TrainEngine(None, max_grad_norm=-1.0)
    with pytest.raises(ValueError, match='max_grad_norm'):
        TrainEngine(None, max_grad_norm=math.nan)
    with pytest.raises(ValueError, match='shard_optimizer'):
        TrainEngine(None, max_grad_norm=1.0, shard_optimizer=True)
    with pytest.raises(ValueError, match='shard_optimizer'):
        Trainer('x', None, None, max_grad_norm=1.0, shard_optimizer=True, world_size=2)


def test_autoencoder_keeps_its_parameters():
    from autolabel_amd.models import Autoencoder
    torch.manual_seed(0)
    a = Autoencoder(32, 8)
    torch.manual_seed(0)
    b = Autoencoder(32, 8, fp8=True)
    assert list(a.state_dict()) == list(b.state_dict())
    assert all(torch.equal(x, y) for x, y in zip(a.state_dict().values(), b.state_dict().values()))
    with pytest.raises(ValueError, match='no CPU path'):
        b(torch.zeros(2, 32))


LINEAR = dict(x=A, x_type=0, ldx=200, fmt_x=0, w=A, ldw=256, sw=A, ldsw=4, fmt_w=0, M=4, N=8, K=200, y=A, ldy=8, y_type=0, relu=0, ws=None, ws_bytes=0, stream=None)
GRAD = dict(g=A, g_type=0, ldg=8, fmt_g=1, x=A, x_type=0, ldx=200, M=1000, N=8, K=200, dw=A, ws=A, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize('bad, match', [
    (dict(x_type=3), 'unknown type'), (dict(y_type=-1), 'unknown type'), (dict(fmt_x=2), 'unknown type'), (dict(fmt_w=-1), 'unknown type'), (dict(M=-1), 'sizes'),
    (dict(M=1 << 31), 'sizes'), (dict(N=0), 'sizes'), (dict(K=0), 'sizes'), (dict(ldy=7), 'sizes'), (dict(ldx=-1), 'sizes'), (dict(ldx=1 << 25), 'sizes'), (dict(ldy=1 << 25), 'sizes'),
    (dict(w=None), '8-bit blocks'), (dict(w=A + 8), '8-bit blocks'), (dict(ldw=128), '8-bit blocks'), (dict(sw=None), '8-bit blocks'), (dict(ldsw=2), '8-bit blocks'),
    (dict(x=None), 'x or y is NULL'), (dict(y=None), 'x or y is NULL'), (dict(x=A + 1), 'not aligned'), (dict(y=A + 2, y_type=2), 'not aligned'),
    (dict(x_type=2), 'workspace'), (dict(x_type=2, ws=A + 8, ws_bytes=1 << 30), 'workspace'), (dict(fmt_w=1, ws=A, ws_bytes=100), 'workspace'),
])
def test_linear_c_refusals(bad, match):
    with pytest.raises(RuntimeError, match=match):
        hip.call('aln_fp8_linear', *{**LINEAR, **bad}.values())


@pytest.mark.parametrize('bad, match', [
    (dict(g_type=3), 'unknown type'), (dict(x_type=-1), 'unknown type'), (dict(fmt_g=2), 'unknown type'), (dict(M=0), 'sizes'), (dict(M=1 << 31), 'sizes'), (dict(N=0), 'sizes'),
    (dict(K=0), 'sizes'), (dict(ldg=7), 'sizes'), (dict(ldx=199), 'sizes'), (dict(ldg=1 << 24), 'sizes'), (dict(ldx=1 << 24), 'sizes'), (dict(g=None), 'NULL'), (dict(x=None), 'NULL'),
    (dict(dw=None), 'NULL'), (dict(g=A + 1), 'not aligned'), (dict(dw=A + 2), 'not aligned'), (dict(ws=None), 'workspace'), (dict(ws_bytes=64), 'workspace'), (dict(ws=A + 4), 'workspace'),
    (dict(g_type=2, ws_bytes=4096), 'workspace'),
])
def test_grad_weight_c_refusals(bad, match):
    with pytest.raises(RuntimeError, match=match):
        hip.call('aln_fp8_grad_weight', *{**GRAD, **bad}.values())


def test_product_workspaces_follow_the_call():
    """No workspace where one launch does it; with one, room for the blocks of x and for the parts of a split contraction."""
    L = hip.lib()
    assert L.aln_fp8_linear_ws_bytes(1 << 20, 4096, 512, 0, 0, 0) == 0 and L.aln_fp8_linear_ws_bytes(1, 4096, 1024, 1, 0, 0) == 0
    for sizes in ((1 << 20, 4096, 512, 2, 0, 0), (1 << 20, 4096, 512, 0, 2, 0), (1 << 20, 4096, 512, 0, 0, 1), (8192, 4096, 1024, 0, 0, 0), (1000, 1000, 1025, 0, 0, 0)):
        m, n, k = sizes[:3]
        assert L.aln_fp8_linear_ws_bytes(*sizes) >= m * -(-k // 128) * 129 + L.aln_fp8_nt_ws_bytes(m, n, k)
    for m, n, k in ((1, 1, 1025), (3, 3304, 1844), (1 << 19, 40, 1203)):        # rows cut on the way: room for parts alone
        assert L.aln_fp8_linear_ws_bytes(m, n, k, 0, 1, 0) % (4 * m * n) == 0
    for m, n, k in ((1, 1, 1), (1003, 130, 77), (1 << 19, 512, 512), (43200, 128, 512)):
        assert L.aln_fp8_grad_weight_ws_bytes(m, n, k, 0, 0) % (4 * n * k) == 0
        assert L.aln_fp8_grad_weight_ws_bytes(m, n, k, 2, 0) >= (n + k) * -(-m // 128) * 129
    assert L.aln_fp8_grad_weight_ws_bytes(0, 5, 5, 0, 0) == 0 and L.aln_fp8_linear_ws_bytes(0, 5, 5, 2, 0, 0) == 0


def test_linear_out_that_autograd_would_miss():
    w = fp8.Fp8Blocks(torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.full((4, 4), 127, dtype=torch.uint8), 100)
    x, out = torch.zeros(3, 100), torch.zeros(3, 4, requires_grad=True)
    with pytest.raises(ValueError, match='must not require a gradient'):
        fp8.linear(x, w, out=out)
    with torch.no_grad(), pytest.raises(ValueError, match='no CPU path'):      # (allowed: it gets as far as the device)
        fp8.linear(x, w, out=out)
