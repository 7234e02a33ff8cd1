"""Results of include/mi_moe_f8.h that would lie in what other blocks of the same launch still read are refused; no GPU needed."""
import ctypes as C

import pytest

from test_layer_host import P, lib, refused  # noqa: F401

Q = P + (1 << 20)  # another place


@pytest.mark.parametrize("drows", ["dout", "rows"])
def test_the_rows_gradient_in_place_of_an_operand(lib, drows):  # noqa: F811
    place = {"dout": Q, "rows": P}[drows]
    refused(lib, "drows", "mi_moe_unsort_tokens_grad", Q, P, P, 0, P, 4, 1, 8, 0, place, P, None)


@pytest.mark.parametrize("name,args", [
    ("mi_moe_sort_tokens", [Q, P, 4, 1, 8, 8, 0, Q, P, P, P, None, 0, None]), ("mi_moe_sort_tokens_grad", [Q, P, 4, 1, 8, 0, Q, None]),
    ("mi_moe_unsort_tokens", [Q, P, 0, P, 4, 1, 8, 0, Q, None])])
def test_rows_in_place_of_tokens(lib, name, args):  # noqa: F811
    refused(lib, "must not be", name, *args)


def test_products_in_place(lib):  # noqa: F811
    n = C.c_size_t()
    assert lib.mi_moe_linear_f8_workspace_size(5, 128, 128, C.byref(n)) == 0
    refused(lib, "y must not be x", "mi_moe_linear_f8", Q, P, P, None, 5, 128, 128, 1, 0, Q, P, n.value, None)
    refused(lib, "y must not be x", "mi_moe_grouped_linear_f8", Q, P, P, P, 5, 2, 128, 128, 1, 0, Q, P, n.value, None)
