"""What surrounds the training operators, on the CPU: waits between launches as the sources have them, states that are saved and go on, gates on several ranks."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _body(source, function):
    text = open(os.path.join(ROOT, "fuselink_b200", "csrc", "kernels", source)).read()
    text = text[text.index("{", text.index(" " + function + "(const")):]
    depth = 0
    for i, c in enumerate(text):
        depth += (c == "{") - (c == "}")
        if depth == 0:
            return text[:i]


def test_every_cta_of_a_kernel_that_starts_early_waits():
    """A CTA that ended without a wait could let what follows begin, and reuse memory, while the kernel in front still works on it."""
    body = _body("losses.cu", "loss_kernel")
    loop, end = body.split("if (policy && threadIdx.x == 0) {")
    assert re.search(r"if \(!asked\) \{\s*asked = true;\s*grid_dep_wait\(\);", loop) and re.search(r"if \(!asked\) grid_dep_wait\(\);", end)
    body = _body("embedding.cu", "embed_sum_kernel")
    assert "return" not in body[:body.index("grid_dep_wait();")]
