"""The operators of a serving step recorded into a graph by the first call of their kind in the process: nothing they need is made
then.  Each runs in a process of its own."""
import pytest

from test_gpu_recorded_first import alone

pytestmark = pytest.mark.gpu

ATTENTION = """
from paged_fixtures import Batch
b = Batch([700, 40 + {new}], [{new}, {new}], 8, 2, 128, 16, seed=1)
want, _ = b.expected()
same = False   # the want is in 64 bits, and a norm cannot tell a weight's rounding from the output's
graph_out = torch.empty_like(b.q)
torch.cuda.synchronize()
with torch.cuda.graph(graph, stream=stream):
    b.run(p, max_new={new}, out=graph_out)
graph.replay()
torch.cuda.synchronize()
from paged_fixtures import held
held(graph_out, *b.expected())
assert torch.equal(b.run(p, max_new={new}), graph_out) and p.device_status() == 0
"""
APPEND = """
from paged_fixtures import Batch, turned
b = Batch([33, 5], [3, 2], 4, 2, 64, 16, seed=1, fill=0.0)
k, v = randn(5, 2, 64), randn(5, 2, 64)
f = p.dispatch.rotary_frequencies(64)
pos = torch.tensor([30, 31, 32, 3, 4], device="cuda")
check(lambda: p.dispatch.paged_append(b.k_pages, b.v_pages, k, v, b.table, b.lens_dev, b.starts, q=b.q, frequencies=f), turned(b.q, pos, f))
"""
ROTARY = """
from paged_fixtures import turned
q, pos, f = randn(5, 4, 64), torch.arange(5, device="cuda"), p.dispatch.rotary_frequencies(64)
check(lambda: p.dispatch.rotary_apply(q, None, pos, f)[0], turned(q, pos, f))
"""
LOGITS = """
z = randn(2, 1000)
ids, values = torch.tensor([[3], [999]], dtype=torch.int32, device="cuda"), torch.tensor([[2.0], [-1.0]], device="cuda")
want = z.double()
want[0, 3] += 2
want[1, 999] -= 1
check(lambda: p.dispatch.adjust_logits(z, bias_ids=ids, bias_values=values), want)
"""


@pytest.mark.parametrize("new", [1, 40])
def test_attention(new):
    alone(ATTENTION.format(new=new))


@pytest.mark.parametrize("code", [APPEND, ROTARY, LOGITS], ids=["append", "rotary", "logits"])
def test_the_others(code):
    alone(code)
