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

    def tiled(x=A, codes=A, affine=A, codes1=None, affine1=None, bias=None, out=A, m=40, n=32, k=512, ldx=512, ldo=32, group=64, act=0, dtype=1, columns=48,
              splits=1, error=A):
        return lib.vx_gemm_q4_tc_shape(x, codes, affine, codes1, affine1, bias, out, m, n, k, ldx, ldo, group, act, dtype, 0, columns, splits, error, None)
    assert tiled(m=0) == 0 and tiled(n=0) == 0
    for change, code in [(dict(columns=8), SHAPE), (dict(columns=40), SHAPE), (dict(columns=272), SHAPE), (dict(columns=144, codes1=A, affine1=A), SHAPE),
                         (dict(splits=0), SHAPE), (dict(splits=9), SHAPE), (dict(splits=5), SHAPE), (dict(error=None), SHAPE), (dict(k=480), SHAPE),
                         (dict(ldx=504), SHAPE), (dict(ldo=16), SHAPE), (dict(codes1=A), SHAPE), (dict(codes1=A, affine1=A, dtype=0), DTYPE),
                         (dict(dtype=3), DTYPE), (dict(ldx=516), ALIGN), (dict(codes=A + 8), ALIGN)]:
        assert tiled(**change) == code, change

    def made(w=A, codes=A, affine=A, n=32, k=128, ldw=128, group=64, dtype=1):
        return lib.vx_quantize_q4(w, codes, affine, n, k, ldw, group, dtype, None)
    assert made(n=0) == 0
    for change, code in [(dict(k=0), SHAPE), (dict(k=96), SHAPE), (dict(group=256), SHAPE), (dict(ldw=64), SHAPE), (dict(dtype=3), DTYPE),
                         (dict(w=A + 2), ALIGN), (dict(ldw=129), ALIGN), (dict(codes=A + 8), ALIGN)]:
        assert made(**change) == code, change
    assert lib.vx_dequantize_q4(A, A, A, 0, 128, 64, None) == 0
    assert lib.vx_dequantize_q4(A, A, A, 32, 96, 64, None) == SHAPE and lib.vx_dequantize_q4(A, A, A + 2, 32, 128, 64, None) == ALIGN


def test_the_entry_points_refuse_sizes_beyond_their_arithmetic():
    """Sizes that cannot be rounded up to a tile within 31 bits, and on the tensor cores depths beyond 2^24."""
    lib = ops.library()
    A, most, deep = 1 << 20, 2 ** 31 - 1, 2 ** 31 - 128

    def product(m, n, k, codes1=None):
        return lib.vx_gemm_q4(A, A, A, codes1, codes1, None, A, m, n, k, k, n, 128, 0, 1, 0, A, None)
    for codes1 in (None, A):
        assert product(1, most, 128, codes1) == LIMIT and product(most, 128, 128, codes1) == LIMIT and product(most, most, 128, codes1) == LIMIT
        assert product(1, 16, deep, codes1) == LIMIT and product(40, 128, deep, codes1) == LIMIT
        assert product(40, 128, (1 << 24) + 128, codes1) == LIMIT
    for m, n, k in [(40, most, 128), (most, 128, 128), (40, 128, deep), (40, 128, (1 << 24) + 128)]:
        assert lib.vx_gemm_q4_tc_shape(A, A, A, None, None, None, A, m, n, k, k, n, 128, 0, 1, 0, 48, 1, A, None) == LIMIT
    for n, k in [(most, 128), (16, deep)]:
        assert lib.vx_quantize_q4(A, A, A, n, k, k, 128, 1, None) == LIMIT
        assert lib.vx_dequantize_q4(A, A, A, n, k, 128, None) == LIMIT


def test_engine_settings():
    from velox_b200 import EngineConfig
    cfg = EngineConfig(weight_bits=4, weight_group=128, head_bits=4)
    assert (cfg.weight_bits, cfg.weight_group, cfg.head_bits) == (4, 128, 4)
    assert EngineConfig().weight_bits is None and EngineConfig().head_bits is None
    for kw, why in [(dict(weight_bits=8), "weight_bits"), (dict(weight_bits=0), "weight_bits"), (dict(head_bits=2), "head_bits"),
                    (dict(weight_bits=4, weight_group=48), "weight_group"), (dict(weight_bits=4, dtype="float32"), "bfloat16"),
                    (dict(head_bits=4, dtype="float32"), "bfloat16")]:
        with pytest.raises(ValueError, match=why):
            EngineConfig(**kw)


def test_which_parts_can_hold_four_bits():
    from helpers import tiny_config
    from velox_b200.config.registry import resolve_architecture
    from velox_b200.models.decoder import DecoderModel
    cfg = tiny_config("tiny_b")
    assert DecoderModel(resolve_architecture(cfg.to_dict()).plan(cfg)).without_four_bits() == []
    from dobepel_helpers import CONFIGS
    raw = CONFIGS["even"]
    arch = resolve_architecture(raw)
    others = DecoderModel(arch.plan(arch.config_class.from_dict(raw))).without_four_bits()
    assert others and "PagedAttention" not in others and "GatedMLP" not in others


def test_rows_that_do_not_go_into_groups_are_named():
    from velox_b200.parts.linear import Linear, linear
    w = torch.zeros(16, 160)
    assert isinstance(linear(w), Linear)
    with pytest.raises(ValueError, match=r"down_proj: rows of 160 do not go into four-bit groups of 64; they go into groups of \[32\]"):
        linear(w, None, 64, "down_proj")
    with pytest.raises(ValueError, match="none of the sizes"):
        linear(torch.zeros(16, 40), None, 32, "w")


def test_the_command_line_names_the_settings():
    from velox_b200.cli import build_parser
    args = build_parser().parse_args(["generate", "--weight-bits", "4", "--weight-group", "128", "--head-bits", "4"])
    assert (args.weight_bits, args.weight_group, args.head_bits) == (4, 128, 4)
    args = build_parser().parse_args(["generate"])
    assert args.weight_bits is None and args.head_bits is None and args.weight_group == 64
    with pytest.raises(SystemExit):
        build_parser().parse_args(["generate", "--weight-bits", "8"])


@pytest.mark.parametrize("rows", [2 ** 31 - 256, 2139095040, 2100000000, 2080374784, 2021195833])
def test_rows_up_to_the_limit_find_a_tile(rows):
    """The tile's choice counts within 31 bits for as many rows as the entry point takes: a refusal (two rounds of tiles too many), not the end of the
    process.  In a process of its own, which a division by zero would end."""
    import subprocess
    import sys
    code = """
from velox_b200.csrc import ops
A = 1 << 20
for codes1 in (None, A):
    print(ops.library().vx_gemm_q4(A, A, A, codes1, codes1, None, A, %d, 256, 64, 64, 256, 64, 0, 1, 0, A, None))
""" % rows
    from helpers import ROOT
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert out.returncode == 0, out.stderr
    assert [int(v) for v in out.stdout.split()] == [LIMIT, LIMIT]


def test_rows_up_to_which_a_matrix_is_streamed():
    few = ops.library().vx_gemm_q4_few_rows
    assert [few(n, k, g) for n, k, g in [(4096, 4096, 0), (4096, 4096, 1), (12288, 4096, 0), (64, 64, 1), (2 ** 31 - 256, 2 ** 31 - 256, 1)]] == [32, 16, 16, 32, 16]
    m = ops.Q4Matrix(*tensors(), 20, 96, 32)
    assert m.few_rows(False) == m.few_rows(True) == 32


def test_a_tied_head_needs_nothing_but_its_table():
    from velox_b200.parts import OutputHead
    head, table = OutputHead("h.", 30, 40, tied=True), torch.zeros(30, 40)
    head.tie(table)
    assert head.weight is table and head.q4 is None
