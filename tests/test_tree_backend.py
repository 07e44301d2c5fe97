"""The attention backend in front of a kernel without the tree form."""

import pytest


def test_a_kernel_without_trees_is_named(pkg):
    class Plain:
        def prefill(self, *args):
            return args

    backend = pkg.AttentionBackend(Plain(), pkg.BackendCapabilities(), {"selected_backend": "plain"})
    with pytest.raises(NotImplementedError, match="plain does not implement draft-tree"):
        backend.tree(1, 2, 3)
    with pytest.raises(NotImplementedError, match="this attention backend"):
        pkg.AttentionBackend(Plain(), pkg.BackendCapabilities(), {}).tree()

    class Tree(Plain):
        def tree(self, *args, window=0):
            return args, window

    assert pkg.AttentionBackend(Tree(), pkg.BackendCapabilities(), {}).tree(1, window=3) == ((1,), 3)
