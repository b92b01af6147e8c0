"""Matrices in four bits: what is refused before anything is launched."""
import pytest
import torch

from velox_b200.csrc import ops


def tensors(rows=20, depth=96, group=32):
    tiles, blocks = -(-rows // 16), -(-depth // 64)
    return torch.zeros(tiles, blocks, 4, 8, 2, 2, dtype=torch.int32), torch.zeros(tiles, blocks * 64 // group, 8, 2, 2, dtype=torch.bfloat16)


def test_a_matrix_holds_tensors_of_its_layout():
    codes, affine = tensors()
    m = ops.Q4Matrix(codes, affine, 20, 96, 32)
    assert m.shape == (20, 96) and m.nbytes == codes.numel() * 4 + affine.numel() * 2 and m.device == codes.device
    for args, why in [((codes, affine, 33, 96, 32), "codes"), ((codes, affine, 20, 160, 32), "codes"), ((codes, affine, 20, 96, 48), "groups of"),
                      ((codes, affine, 20, 96, 64), "multiple of the group"), ((codes, affine, 20, 100, 32), "multiple of the group"),
                      ((codes.to(torch.int64), affine, 20, 96, 32), "int32"), ((codes, affine.float(), 20, 96, 32), "bfloat16"),
                      ((codes, affine[:, :2], 20, 96, 32), "offsets"), ((codes.transpose(2, 3).contiguous().transpose(2, 3), affine, 20, 96, 32), "contiguous"),
                      ((codes, affine, 0, 96, 32), "positive"), ((codes, affine, 20, 0, 32), "positive")]:
        with pytest.raises(ops.KernelError, match=why):
            ops.Q4Matrix(*args)


def test_operators_take_cuda_tensors_only():
    m = ops.Q4Matrix(*tensors(), 20, 96, 32)
    x = torch.zeros(2, 96, dtype=torch.bfloat16)
    for call in (lambda: ops.gemm_q4(x, m), lambda: ops.gated_q4(x, m, m), lambda: ops.quantize_q4(x, 32), lambda: ops.dequantize_q4(m)):
        with pytest.raises(ops.KernelError, match="CUDA tensors"):
            call()


SHAPE, DTYPE, ALIGN, LIMIT = -1, -2, -3, -4


def test_the_entry_points_refuse_before_they_launch():
    """Sizes, types and alignment are refused by the C entry points themselves; nothing to do is no error.  (No address here is read.)"""
    lib = ops.library()
    A = 1 << 20

    def product(x=A, codes=A, affine=A, codes1=None, affine1=None, bias=None, out=A, m=2, n=32, k=128, ldx=128, ldo=32, group=64, act=0, dtype=1):
        return lib.vx_gemm_q4(x, codes, affine, codes1, affine1, bias, out, m, n, k, ldx, ldo, group, act, dtype, 0, A, None)
    assert product(m=0) == 0 and product(n=0) == 0
    for change, code in [(dict(k=0), SHAPE), (dict(k=96), SHAPE), (dict(group=16), SHAPE), (dict(ldx=120), SHAPE), (dict(ldo=31), SHAPE),
                         (dict(codes1=A), SHAPE), (dict(codes1=A, affine1=A, bias=A), SHAPE), (dict(codes1=A, affine1=A, act=6), SHAPE),
                         (dict(codes1=A, affine1=A, act=-1), SHAPE), (dict(ldx=132), ALIGN), (dict(x=A + 8), ALIGN), (dict(codes=A + 4), ALIGN),
                         (dict(affine=A + 4), ALIGN), (dict(codes1=A + 4, affine1=A), ALIGN), (dict(dtype=2), DTYPE), (dict(dtype=-1), DTYPE),
                         (dict(codes1=A, affine1=A, dtype=0), DTYPE)]:
        assert product(**change) == code, change

    def made(w=A, codes=A, affine=A, n=32, k=128, ldw=128, group=64, dtype=1):
        return lib.vx_quantize_q4(w, codes, affine, n, k, ldw, group, dtype, None)
    assert made(n=0) == 0
    for change, code in [(dict(k=0), SHAPE), (dict(k=96), SHAPE), (dict(group=256), SHAPE), (dict(ldw=64), SHAPE), (dict(dtype=3), DTYPE),
                         (dict(w=A + 2), ALIGN), (dict(ldw=129), ALIGN), (dict(codes=A + 8), ALIGN)]:
        assert made(**change) == code, change
    assert lib.vx_dequantize_q4(A, A, A, 0, 128, 64, None) == 0
    assert lib.vx_dequantize_q4(A, A, A, 32, 96, 64, None) == SHAPE and lib.vx_dequantize_q4(A, A, A + 2, 32, 128, 64, None) == ALIGN
