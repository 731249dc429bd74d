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
