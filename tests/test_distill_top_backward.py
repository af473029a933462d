"""The gradient Function of top_kl_loss can be run directly in a plain backward pass (linear.apply_in_backward)."""
import ast
import inspect
import textwrap

from sparseforge_amd import distill, distill_top, linear


def test_forward_asks_its_ctx_for_no_more_than_the_stand_in_has():
    tree = ast.parse(textwrap.dedent(inspect.getsource(distill_top._TopKLGrad.forward)))
    loads = {n.attr for n in ast.walk(tree) if isinstance(n, ast.Attribute) and isinstance(n.ctx, ast.Load)
             and isinstance(n.value, ast.Name) and n.value.id == "ctx"}
    assert loads <= {name for name in vars(linear._Unrecorded) if not name.startswith("__")}


def test_reached_from_distill():
    for name in ("TopLogits", "top_logits", "top_kl_loss"):
        assert getattr(distill, name) is getattr(distill_top, name)
