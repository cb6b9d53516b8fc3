"""The tile kernels with a fused epilogue keep their accumulators in registers that the compiler does not know of and load tiles by
instructions that it does not know either, as the kernels without one: what it makes around them, looked at in the assembly
(cross-compiled, no GPU)."""

import itertools
import os
import re
import shutil
import subprocess

import pytest

from msamp import _backend

TYPES = ('float', 'f16_t', 'bf16_t')    # the three translation units of the Makefile


@pytest.fixture(scope='module')
def assembly(tmp_path_factory):
    """{type: {kernel: [(inside inline assembly, instruction)]}}"""
    hipcc = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'
    if not os.path.exists(hipcc):
        pytest.skip('no hipcc here')
    src = os.path.join(os.path.dirname(_backend.__file__), '..', 'csrc')
    tmp = tmp_path_factory.mktemp('fused_asm')
    procs = []
    for name in TYPES:
        out = str(tmp / f'{name}.s')
        cmd = [hipcc, '--offload-arch=gfx950', '-O3', '-std=c++17', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
               '-Wno-unused-command-line-argument', '-Wno-inline-asm', f'-DMSAMP_FUSED_OT={name}', '--cuda-device-only', '-S', '-o', out,
               os.path.join(src, 'gemm_fused_tiles.hip')]
        procs.append((name, out, subprocess.Popen(cmd, cwd=src, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    found = {}
    for name, out, proc in procs:
        log = proc.communicate()[0]
        assert proc.returncode == 0, log.decode(errors='replace')[-2000:]
        kernels, kernel, in_asm = {}, None, False
        for line in open(out):
            m = re.match(r'^(_Z\w+):', line)
            if m:
                kernel = m.group(1)
            in_asm = (in_asm or '#ASMSTART' in line) and '#ASMEND' not in line
            code = line.split(';')[0].strip()
            if not m and kernel and code and not code.startswith(('.', '#')) and not code.endswith(':'):
                kernels.setdefault(kernel, []).append((in_asm, code))
        found[name] = kernels
    return found


def registers(kind, text):
    """Numbers of the vector (v), scalar (s) or accumulation (a) registers that an instruction names."""
    return {n for m in re.finditer(r'\b%s(\d+)\b|\b%s\[(\d+):(\d+)\]' % (kind, kind), text)
            for n in ([int(m.group(1))] if m.group(1) else range(int(m.group(2)), int(m.group(3)) + 1))}


@pytest.mark.parametrize('name', TYPES)
def test_compiler_leaves_the_accumulators_alone(assembly, name):
    counts = {}
    for kernel, lines in assembly[name].items():
        form = next((f for f in ('fp8_gemm_dma_fused_kernel', 'fp8_gemm_dma128_fused_kernel', 'fp8_gemm_pair128_fused_kernel') if f in kernel), None)
        assert form is not None, kernel
        counts[form] = counts.get(form, 0) + 1
        assert not any(code.startswith('scratch_') for _, code in lines), kernel    # (a reload waits for the tile loads in flight)
        outside = [code for in_asm, code in lines if not in_asm]
        if 'pair128' in form:    # accumulators from v192 on
            assert max((max(registers('v', code), default=0) for code in outside)) < 192, kernel
        else:    # all accumulation registers
            assert not any(registers('a', code) for code in outside), kernel
    assert counts == {f: 2 for f in counts} and len(counts) == 3    # whole slices of K and a ragged last one


@pytest.mark.parametrize('name', TYPES)
def test_operands_and_addresses_are_there_in_time(assembly, name):
    """No vector instruction writes an operand of an MFMA less than two instructions ahead of it; a load to LDS has a wait state behind
    the instruction that writes M0, and five behind a vector instruction that writes its scalar base."""
    for kernel, lines in assembly[name].items():
        products, loads, recent, m0, vector = 0, 0, [], 9, {}
        for in_asm, code in lines:
            op, args = code.split()[0], code[len(code.split()[0]):].split(',')
            if op.startswith('v_mfma'):
                products += 1
                assert not (registers('v', args[1]) | registers('v', args[2])) & set().union(*recent[-2:]), (kernel, code)
            if '_load_lds_' in op:
                loads += 1
                assert m0 >= 1 and all(vector.get(r, 9) >= 5 for r in registers('s', args[-1])), (kernel, code)
            states = int(args[0], 0) + 1 if op == 's_nop' else 1
            recent += [set()] * states if op == 's_nop' else [registers('v', args[0]) if op.startswith('v_') and 'mfma' not in op else set()]
            recent = recent[-2:]
            m0, vector = m0 + states, {r: n + states for r, n in vector.items() if n < 9}
            if args[0].strip() == 'm0':
                m0 = 0
            elif op.startswith('v_'):
                vector.update((r, 0) for r in registers('s', args[0]))
        assert products >= 16 and loads >= 16, kernel


@pytest.mark.parametrize('name', TYPES)
def test_accumulators_are_read_behind_the_products(assembly, name):
    """The stores of accumulators to LDS come behind the wait for the last product: no MFMA follows one of them before the kernel's end,
    and between the last MFMA and the first of them lie the wait states that the result takes."""
    for kernel, lines in assembly[name].items():
        if 'fp8_gemm_dma_fused_kernel' not in kernel:
            continue
        codes = [code for _, code in lines]
        stores = [i for i, code in enumerate(codes) if code.startswith('ds_write_b128') and registers('a', code)]
        last = max(i for i, code in enumerate(codes) if code.startswith('v_mfma'))
        assert len(stores) >= 64 and min(stores) > last
        states = sum(int(code.split()[1], 0) + 1 if code.startswith('s_nop') else 1 for code in codes[last + 1:min(stores)])
        assert states >= 20, (kernel, states)


def test_every_kernel_is_looked_at(assembly):
    assert len(set(itertools.chain.from_iterable(assembly.values()))) == 18


def test_output_may_be_the_residual(tmp_path):
    """The fused forms promise the compiler nothing about what else points to their output; the others, whose outputs are their own, do."""
    hipcc = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'
    if not os.path.exists(hipcc):
        pytest.skip('no hipcc here')
    src = os.path.join(os.path.dirname(_backend.__file__), '..', 'csrc')
    common = [hipcc, '--offload-arch=gfx950', '-O3', '-std=c++17', '-Wno-unused-command-line-argument', '-Wno-inline-asm', '--cuda-device-only', '-S', '-emit-llvm',
              '-Xclang', '-disable-llvm-passes']
    seen = set()
    for unit, defines in (('gemm_fused_tiles', ['-DMSAMP_FUSED_OT=bf16_t']), ('gemm_inst', ['-DMSAMP_XF=5', '-DMSAMP_YF=5'])):
        out = str(tmp_path / f'{unit}.ll')
        done = subprocess.run([*common, *defines, '-o', out, os.path.join(src, unit + '.hip')], cwd=src, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
        assert done.returncode == 0, done.stdout.decode(errors='replace')[-2000:]
        for line in open(out):
            m = re.match(r'define .*@(_ZN5msamp11gemm_dma(?:256|128)I\w+)\(([^)]*)\)', line)
            if not m:
                continue
            x, y, d = m.group(2).split(', ')[:3]
            fused = unit == 'gemm_fused_tiles'
            assert 'noalias' in x and 'noalias' in y and ('noalias' in d) != fused, (m.group(1), d)
            seen.add((unit, 'dma256' in m.group(1)))
    assert ('gemm_fused_tiles', True) in seen and ('gemm_fused_tiles', False) in seen and ('gemm_inst', True) in seen
