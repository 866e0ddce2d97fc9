"""How the library cuts a call of the training operators: csrc/linear_plan.h built into a small host program (tests/c/linear_plan.cpp)."""
import functools
import json
import os
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODES = {'fp32': 0, 'bf16': 1, 'fp16': 2}
ACTS = {'none': 0, 'relu': 1, 'leaky_relu': 2, 'sigmoid': 3, 'tanh': 4, 'gelu': 5, 'silu': 6}


@functools.lru_cache(None)
def _program():
    path = os.path.join(tempfile.mkdtemp(prefix='linear_plan_'), 'linear_plan')
    subprocess.check_call(['g++', '-std=c++17', '-O1', '-Wall', '-Werror', '-D__HIP_PLATFORM_AMD__', '-isystem', '/opt/rocm/include', '-I',
                           os.path.join(ROOT, 'rgb-d-pifuhd_amd', 'csrc'), os.path.join(ROOT, 'tests', 'c', 'linear_plan.cpp'), '-o', path])
    return path


def ask(line):
    out = subprocess.run([_program()], input=line + '\n', capture_output=True, text=True, check=True).stdout
    return json.loads(out)


def product(elem, I, J, P, a_dma=True, b_dma=True):     # noqa: E741
    return ask(f'product {elem} {I} {J} {P} {int(a_dma)} {int(b_dma)}')['product']


def forward(dtype, m, n, k, ldx=None, ldw=None):
    return ask(f'forward {CODES[dtype]} {m} {n} {k} {ldx or k} {ldw or k}')


def backward(dtype, m, n, k, act='none', x_act='none', packed=False, ldg=None, ldx=None, ldw=None, need=('x', 'weight', 'bias')):
    gradients = sum(v for name, v in (('x', 1), ('weight', 2), ('bias', 4)) if name in need)
    return ask(f'backward {CODES[dtype]} {ACTS[act]} {ACTS[x_act]} {int(packed)} {m} {n} {k} {ldg or n} {ldx or k} {ldw or k} {gradients}')


def expect(plan, **cut):
    """Fails where a product is no longer cut as its test was written for: such a test needs another size, not another tolerance."""
    got = {name: plan[name] for name in cut}
    if got != cut:
        pytest.fail(f'cut {plan}, the test is for {cut}')
