"""Every test that a module defines is collected: a second definition of a name takes the first one's place without a word."""
import ast
import glob
import os

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def lost_tests(source):
    """Tests whose name is bound again later, and that no other name was given before that."""
    bound, kept, lost = set(), set(), []
    for node in ast.parse(source).body:
        if isinstance(node, ast.Assign) and isinstance(node.value, ast.Name) and any(isinstance(t, ast.Name) and t.id.startswith("test_") for t in node.targets):
            kept.add(node.value.id)
        if isinstance(node, (ast.FunctionDef, ast.ClassDef)) and node.name.lower().startswith("test"):
            if node.name in bound and node.name not in kept:
                lost.append(node.name)
            bound.add(node.name)
            kept.discard(node.name)
    return lost


def test_what_is_lost():
    one, two = "def test_a(): pass\n", "def test_a(x): pass\n"
    assert lost_tests(one + two) == ["test_a"]
    assert lost_tests(one + "test_b = test_a\n" + two) == []
    assert lost_tests(one + "test_b = test_a\n" + two + one) == ["test_a"]
    assert lost_tests(one + "def test_b(): pass\n") == []


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(HERE, "test_*.py"))), ids=os.path.basename)
def test_no_test_is_lost(path):
    with open(path) as f:
        assert lost_tests(f.read()) == []
