"""What the operators over large item vocabularies refuse, decided before anything reaches a GPU: the C entries' checks of sizes, types,
pointers and alignment, and the Python wrappers' of devices, types and shapes."""
import ctypes

import pytest
import torch

OK, EINVAL, ESHAPE, EUNSUPPORTED = 0, -1, -4, -6
P = ctypes.c_void_p
A, B, C, D, W = P(1 << 20), P(2 << 20), P(3 << 20), P(4 << 20), P(5 << 20)  # never dereferenced: every call below ends in a check


def embedding(lib, table=A, ldt=8, rows=4, d=8, dtype=0, ids=B, n=3, out=C, ldo=8):
    return lib.rbg_embedding(table, ldt, rows, d, dtype, ids, n, 1.0, out, ldo, None)


def embedding_grad(lib, grad=A, ldg=8, dtype=1, ids=B, n=3, rows=4, d=8, out=C, out_dtype=1, work=W):
    return lib.rbg_embedding_grad(grad, ldg, dtype, ids, n, rows, d, 1.0, -1, out, out_dtype, work, None)


def distill(lib, z=A, ldz=8, dtype=0, n=2, v=8, idx=B, val=C, k=2, t=1.0, loss=D, grad=None, ldg=8, work=W):
    return lib.rbg_distill_topk(z, ldz, dtype, n, v, idx, val, k, t, None, loss, None, grad, ldg, work, None)


def logp(lib, z=A, ldz=8, dtype=0, m=2, v=8, targets=B, out=C, work=W):
    return lib.rbg_token_logp(z, ldz, dtype, m, v, targets, out, None, work, None)


def preference(lib, z=A, ldz=8, dtype=0, m=2, v=8, targets=B, offsets=B, pairs=1, ref=C, beta=0.1, smoothing=0.0, loss=D, margin=D, grad=P(6 << 20), ldg=8,
               work=W):
    return lib.rbg_preference_grad(z, ldz, dtype, m, v, targets, offsets, pairs, ref, beta, smoothing, None, loss, margin, grad, ldg, work, None)


def quantize(lib, x=A, ldx=8, dtype=0, n=2, k=8, codes=B, ldc=16, scale=C):
    return lib.rbg_quantize_rows_i8(x, ldx, dtype, n, k, codes, ldc, scale, None)


def score(lib, qu=A, ldu=128, su=B, b=2, qi=C, ldi=16, si=B, n=3, k=8, s=D, lds=3, out=0):
    return lib.rbg_score_i8(qu, ldu, su, b, qi, ldi, si, n, k, s, lds, out, None)


def score_rows(lib, u=A, ldu=8, dtype=0, b=2, qi=C, ldi=16, si=B, n=3, k=8, s=D, lds=3, out=0, work=W):
    return lib.rbg_score_rows_i8(u, ldu, dtype, b, qi, ldi, si, n, k, s, lds, out, work, None)


REFUSED = [
    (embedding, dict(dtype=3), EINVAL), (embedding, dict(d=0), ESHAPE), (embedding, dict(ldt=7), ESHAPE), (embedding, dict(ldo=7), ESHAPE),
    (embedding, dict(n=-1), ESHAPE), (embedding, dict(ids=None), EINVAL), (embedding, dict(table=None), EINVAL), (embedding, dict(out=P(2)), EINVAL), (embedding, dict(n=(1 << 34) + 1), EUNSUPPORTED),
    (embedding_grad, dict(out_dtype=2), EINVAL), (embedding_grad, dict(ldg=7), ESHAPE), (embedding_grad, dict(rows=0x7fffffff), EUNSUPPORTED),
    (embedding_grad, dict(n=0x7fff0000), EUNSUPPORTED), (embedding_grad, dict(d=(1 << 20) + 1, ldg=1 << 21), EUNSUPPORTED), (embedding_grad, dict(work=P(8)), EINVAL),
    (embedding_grad, dict(work=None, n=1000), EINVAL), (embedding_grad, dict(grad=P(1)), EINVAL),
    (distill, dict(k=0), EUNSUPPORTED), (distill, dict(k=257), EUNSUPPORTED), (distill, dict(t=0.0), EINVAL), (distill, dict(t=float("nan")), EINVAL),
    (distill, dict(t=-1.0), EINVAL), (distill, dict(v=0), ESHAPE), (distill, dict(ldz=7), ESHAPE), (distill, dict(dtype=-1), EINVAL),
    (distill, dict(z=P(2)), EINVAL), (distill, dict(loss=None), EINVAL), (distill, dict(work=P(4)), EINVAL), (distill, dict(grad=P((1 << 20) + 32)), EINVAL),
    (distill, dict(grad=A, ldg=9), EINVAL), (distill, dict(grad=D, ldg=7), ESHAPE), (distill, dict(v=1 << 31, ldz=1 << 31), EUNSUPPORTED),
    (logp, dict(targets=None), EINVAL), (logp, dict(v=-1), ESHAPE), (logp, dict(work=None, v=50000, ldz=50000), EINVAL), (distill, dict(work=None, v=50000, ldz=50000), EINVAL),
    (preference, dict(beta=float("inf")), EINVAL), (preference, dict(smoothing=-0.1), EINVAL), (preference, dict(smoothing=1.5), EINVAL),
    (preference, dict(smoothing=float("nan")), EINVAL), (preference, dict(offsets=None), EINVAL), (preference, dict(pairs=-1), ESHAPE),
    (preference, dict(ref=None), EINVAL), (preference, dict(grad=None), EINVAL), (preference, dict(grad=P((1 << 20) - 32)), EINVAL),
    (quantize, dict(ldc=24), EINVAL), (quantize, dict(ldc=0), ESHAPE), (quantize, dict(codes=P(8)), EINVAL), (quantize, dict(k=0), ESHAPE),
    (quantize, dict(x=P(2)), EINVAL), (quantize, dict(scale=None), EINVAL),
    (score, dict(ldu=64), EINVAL), (score, dict(ldi=24), EINVAL), (score, dict(k=131072, ldu=131072, ldi=131072), EUNSUPPORTED), (score, dict(lds=2), ESHAPE), (score, dict(ldi=(1 << 23) + 16), EUNSUPPORTED), (score, dict(ldu=(1 << 23) + 128), EUNSUPPORTED),
    (score, dict(qi=P(8)), EINVAL), (score, dict(out=3), EINVAL), (score, dict(k=0), ESHAPE), (score, dict(su=None), EINVAL),
    (score_rows, dict(dtype=3), EINVAL), (score_rows, dict(out=-1), EINVAL), (score_rows, dict(ldu=7), ESHAPE), (score_rows, dict(work=None), EINVAL),
    (score_rows, dict(work=P(8)), EINVAL), (score_rows, dict(u=P(2)), EINVAL), (score_rows, dict(k=131072, ldu=131072, ldi=131072), EUNSUPPORTED),
    (score_rows, dict(lds=2), ESHAPE), (score_rows, dict(n=1 << 31, lds=1 << 31), EUNSUPPORTED), (score_rows, dict(k=0), ESHAPE),
]


@pytest.mark.parametrize("call,args,code", REFUSED, ids=[f"{c.__name__}-{'-'.join(a)}" + f"-{i}" for i, (c, a, _) in enumerate(REFUSED)])
def test_c_entries_refuse(rbg, call, args, code):
    assert call(rbg._lib.lib, **args) == code
    assert rbg._lib.lib.rbg_last_error()


def test_nothing_to_do_is_no_error(rbg):
    lib = rbg._lib.lib
    assert embedding(lib, n=0, ids=None, out=None) == OK
    assert embedding_grad(lib, rows=0) == OK
    assert distill(lib, n=0, z=None) == OK
    assert logp(lib, m=0, z=None) == OK
    assert preference(lib, m=0, pairs=0, z=None) == OK
    assert quantize(lib, n=0) == OK and score(lib, b=0) == OK and score(lib, n=0, lds=0) == OK and score_rows(lib, b=0) == OK
    assert lib.rbg_preference_loss(None, 0, A, 0, None, 0.1, 0.0, None, None, None) == OK


def test_workspaces(rbg):
    lib, n = rbg._lib.lib, ctypes.c_int64()
    for fn, args in ((lib.rbg_embedding_grad_workspace, (500, 7, 8)), (lib.rbg_embedding_grad_workspace, (100000, 7, 8)), (lib.rbg_distill_topk_workspace, (3, 50000)),
                     (lib.rbg_token_logp_workspace, (3, 50000)), (lib.rbg_score_rows_i8_workspace, (3, 500)), (lib.rbg_preference_grad_workspace, (3, 50000))):
        assert fn(*args, ctypes.byref(n)) == OK and n.value > 0 and n.value % 16 == 0
        assert fn(*args, None) == EINVAL
        assert fn(-1, *args[1:], ctypes.byref(n)) == ESHAPE


def test_wrappers_refuse_the_cpu(rbg):
    f, i = torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: rbg.embedding(f, i), lambda: rbg.embedding_grad(f, i, 3), lambda: rbg.distill_topk(f, i[:, None], f[:, :1]),
                 lambda: rbg.distill_topk_grad(f, i[:, None], f[:, :1]), lambda: rbg.token_logp(f, i), lambda: rbg.preference_loss(f[0], i, f[0]),
                 lambda: rbg.preference_grad(f, i, i, f[0]), lambda: rbg.quantize_rows(f), lambda: rbg.score_int8(f, i, i)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@pytest.mark.parametrize("d", [(1 << 30) + 1, (1 << 31) - 1])
def test_lookup_refuses_columns_that_its_steps_would_pass(rbg, d):
    """A kernel's column steps past d by up to 512 elements in 32 bits."""
    assert embedding(rbg._lib.lib, d=d, ldt=d, ldo=d) == EUNSUPPORTED


def test_sizes_that_32_bits_would_cut_are_refused(rbg):
    assert rbg.vocab._c_int(0x7fffffff, "d") == 0x7fffffff
    with pytest.raises(ValueError, match="k = 4294967297"):
        rbg.vocab._teacher(torch.empty(1, 4), torch.zeros(1, 1, dtype=torch.int64).expand(1, (1 << 32) + 1), torch.zeros(1, 1).expand(1, (1 << 32) + 1))
    with pytest.raises(ValueError, match="columns of table"):
        rbg.vocab._embedding(torch.empty(1, (1 << 32) + 8, device="meta"), torch.zeros(3, dtype=torch.int64), 1.0)
