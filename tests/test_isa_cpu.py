"""tools/isa_mfma_lint.py -- the wait states between matrix instructions and what touches their results, counted in the code that was built -- on planted
sequences, and on the 8-bit kernels of the built library."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location('isa_mfma_lint', os.path.join(ROOT, 'tools', 'isa_mfma_lint.py'))
L = importlib.util.module_from_spec(spec)
spec.loader.exec_module(L)

PRODUCT = 'v_mfma_i32_32x32x32_i8 v[0:15], v[20:23], v[24:27], v[0:15]'
READ = 'v_cvt_f32_i32_e32 v30, v3'


def listing(lines):
    """llvm-objdump's form: eight bytes an instruction; '@n' names the branch target n."""
    out = ['0000000000001000 <kernel>:']
    for i, line in enumerate(lines):
        text, _, target = line.partition(' @')
        out.append(f'\t{text:60s}// {0x1000 + 8 * i:012X}: 00000000 00000000' + (f' <kernel+0x{8 * int(target):x}>' if target else ''))
    return '\n'.join(out)


def found(*lines):
    return [(d, n) for d, n, _, _ in L.lint(L.parse(listing(lines))['kernel'])[0]]


def test_planted_sequences():
    assert found(PRODUCT, READ) == [(0, 12)]
    assert found(PRODUCT, 's_nop 10', READ) == [(11, 12)]
    assert found(PRODUCT, 's_nop 11', READ) == []
    assert found(PRODUCT, 's_nop 15', READ) == []
    # on the far side of a branch that is taken, with enough on the near side
    assert found(PRODUCT, 's_cbranch_scc1 2 @4', 's_nop 15', READ, 's_nop 2', READ, 's_endpgm') == [(4, 12)]
    assert found(PRODUCT, 's_branch 2 @4', READ, 's_endpgm', 's_nop 10', READ, 's_endpgm') == []
    # behind the back edge of a loop
    assert found('v_mov_b32_e32 v40, v3', 's_nop 15', PRODUCT, 's_cbranch_scc1 65532 @0', 's_nop 15', READ) == [(1, 12)]
    # an accumulation may follow at once, a product that multiplies the result or takes a part of it may not; a write is a touch too
    assert found(PRODUCT, PRODUCT, 's_nop 15', READ) == []
    assert found(PRODUCT, 'v_mfma_i32_32x32x32_i8 v[40:55], v[20:23], v[24:27], v[0:15]', 's_nop 15', READ) == []
    assert found(PRODUCT, 'v_mfma_i32_32x32x32_i8 v[40:55], v[0:3], v[24:27], v[40:55]', 's_nop 15') == [(0, 12)]
    assert found(PRODUCT, 'v_mfma_i32_16x16x64_i8 v[40:43], v[20:23], v[24:27], v[4:7]', 's_nop 15') == [(0, 12)]
    assert found(PRODUCT, 's_nop 3', 'v_mov_b32_e32 v15, 0') == [(4, 12)]
    assert found('v_mfma_i32_16x16x64_i8 a[0:3], v[20:23], v[24:27], a[0:3]', 's_nop 5', 'v_accvgpr_read_b32 v0, a2') == [(6, 8)]
    assert found('v_mfma_i32_16x16x64_i8 a[0:3], v[20:23], v[24:27], a[0:3]', 's_nop 5', 'v_mov_b32_e32 v0, v2') == []


@pytest.mark.skipif(not os.path.exists(L.OBJDUMP), reason='needs llvm-objdump')
def test_built_kernels_leave_results_alone(built_lib):
    from edgegan_amd import _lib
    kernels = L.parse(L.disassemble(_lib.LIB_PATH))
    products = {name: code for name, code in kernels.items() if any(op.startswith('v_mfma') and L.shape(op) in L.NEEDED for op, _, _ in code)}
    assert sum('int8_' in name for name in products) >= 30
    for name, code in products.items():
        bad, _ = L.lint(code)
        assert not bad, (name, [(d, n, code[p], code[q]) for d, n, p, q in bad])
