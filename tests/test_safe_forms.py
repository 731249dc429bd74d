"""Forms that the card's software does not carry safely stay out of the package (CPU: they are found by reading the sources and the build)."""
import ast
import os

ROOT = os.path.join(os.path.dirname(__file__), '..')


def _python_sources():
    yield os.path.join(ROOT, 'bench.py')
    for folder, _, names in os.walk(os.path.join(ROOT, 'pseldnets_amd')):
        for n in names:
            if n.endswith('.py'):
                yield os.path.join(folder, n)


def test_every_stream_has_the_default_priority():
    """Work on streams of different priorities can hang the GPU: no stream and no process group asks for another than the default."""
    for path in _python_sources():
        with open(path) as f:
            tree = ast.parse(f.read())
        for call in ast.walk(tree):
            if not isinstance(call, ast.Call):
                continue
            for kw in call.keywords:
                if kw.arg in ('priority', 'is_high_priority_stream'):
                    assert isinstance(kw.value, ast.Constant) and not kw.value.value, f'{path}:{call.lineno}'
            if isinstance(call.func, ast.Attribute) and call.func.attr == 'Stream':
                assert len(call.args) < 2, f'{path}:{call.lineno}'      # (the second positional argument is the priority)
    for folder, _, names in os.walk(os.path.join(ROOT, 'pseldnets_amd', 'csrc')):
        for n in names:
            if n.endswith(('.hip', '.h', '.cpp')):
                with open(os.path.join(folder, n)) as f:
                    assert 'StreamCreateWithPriority' not in f.read(), n


def test_no_packed_fp32_instruction_is_written_or_built():
    """Some operand-select forms of the packed fp32 instructions can give wrong results: no source writes one, and every HIP compilation forbids the
    compiler to form them."""
    import shutil
    import subprocess
    csrc = os.path.join(ROOT, 'pseldnets_amd', 'csrc')
    for folder, _, names in os.walk(csrc):
        for n in names:
            if n.endswith(('.hip', '.h')):
                with open(os.path.join(folder, n)) as f:
                    text = f.read()
                for form in ('v_pk_add_f32', 'v_pk_mul_f32', 'v_pk_fma_f32'):
                    assert form not in text, (n, form)
    assert shutil.which('make')
    plan = subprocess.run(['make', '-n', '-B', '-C', csrc], check=True, capture_output=True, text=True).stdout
    compiled = [line for line in plan.splitlines() if 'hipcc' in line and '.hip' in line]
    assert len(compiled) >= 22
    for line in compiled:
        assert '-Xclang -target-feature -Xclang -packed-fp32-ops' in line, line
