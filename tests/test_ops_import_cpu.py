"""The package's names without torch: only the calls that take tensors need it."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(code):
    out = subprocess.run([sys.executable, '-c', 'import sys\nsys.path.insert(0, %r)\n' % ROOT + code],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    return out.stdout


def test_all_names_without_torch():
    out = run('''
sys.modules['torch'] = None          # an import of torch raises ImportError
from pgvector_b200 import *
import pgvector_b200 as pb
assert softmax_loss is pb.softmax_loss and matmul_blocks is pb.matmul_blocks and Shard is pb.Shard
for name in pb.__all__:
    getattr(pb, name)
for f in (softmax_loss, softmax_loss_grad, quantize_blocks, matmul_blocks):
    try:
        f(*[None] * 4) if f is not quantize_blocks else f(None)
    except ImportError:
        print('needs torch')
''')
    assert out.count('needs torch') == 4


def test_names_do_not_import_torch():
    run('''
from pgvector_b200 import *
assert 'torch' not in sys.modules
import inspect
assert 'targets' in inspect.signature(softmax_loss).parameters and quantize_blocks.__doc__
''')


def test_operands_that_need_a_gradient_are_checked_first():
    run('''
import torch
import pgvector_b200 as pb
x, t = torch.zeros(4, 8, requires_grad=True), torch.zeros(4, dtype=torch.int64)
try:
    pb.softmax_loss(x, x, t)
    raise SystemExit('taken')
except pb.AnnB200Error as e:
    assert e.status == pb.INVALID
''')
