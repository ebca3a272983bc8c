"""Sizes at which the tensor-core kernel takes each of its forms on a GPU of 148 multiprocessors: shared by the CPU test that
they do and the GPU tests of their results.  Odd sizes, so that tiles are ragged and operands are copied."""

SMS = 148
# (rows, inner, outer): tile width, blocks that share a tile's sums, pairs
FORWARD = {
    (72, 17, 16): (64, 1, 0), (396, 2803, 593): (64, 2, 0), (66, 2206, 16): (64, 4, 0), (69, 3872, 18): (64, 8, 0),
    (134, 21, 4752): (128, 1, 0), (807, 5325, 690): (128, 2, 0), (386, 5685, 592): (128, 4, 0),
    (262, 22, 6394): (256, 1, 0), (2214, 219, 1540): (256, 1, 1),
    # few rows on the tiles' narrow side
    (5, 64, 130): (64, 1, 0), (5, 2646, 4872): (64, 2, 0), (7, 2240, 30): (64, 4, 0), (9, 3968, 24): (64, 8, 0), (64, 80, 20000): (64, 1, 0),
    # several tiles to a block: the bias and the residual of the next are fetched under the products of this one
    (6288, 21, 268): (64, 1, 0), (2080, 539, 1671): (128, 1, 0), (2053, 22, 6117): (256, 1, 0), (2587, 721, 2720): (256, 1, 1),
    (4100, 1000, 4104): (256, 1, 1),
}
# a backward pass: each of its launches; one launch forms both products
BACKWARD = {
    (3, 16, 18): [(64, 1, 0)], (139, 4879, 134): [(64, 1, 0)], (4, 324, 3001): [(64, 1, 0)],
    (3, 4907, 16): [(128, 1, 0)], (529, 4310, 528): [(128, 1, 0)], (678, 1376, 1487): [(128, 1, 0)], (1521, 3100, 663): [(128, 1, 0)],
    (129, 7804, 139): [(256, 1, 0)], (526, 8875, 614): [(256, 1, 0)], (1532, 7675, 552): [(256, 1, 0)],
    (132, 8294, 203): [(256, 1, 1)], (904, 6300, 645): [(256, 1, 1)], (1700, 2951, 768): [(256, 1, 1)], (1644, 4817, 796): [(256, 1, 1)],
    (4434, 222, 519): [(64, 4, 0), (64, 1, 0)], (2659, 23, 8138): [(64, 4, 0), (64, 2, 0)], (4, 131, 6439): [(64, 8, 0), (128, 1, 0)],
    (5756, 585, 150): [(64, 4, 0), (256, 1, 0)], (205, 584, 5921): [(64, 4, 0), (256, 1, 1)], (7836, 488, 515): [(128, 4, 0), (128, 1, 0)],
}


def shapes(lib, sms, size, backward):
    import ctypes as C

    a = (C.c_int32 * 7)()
    assert lib.fv_linear_shapes(sms, *size, int(backward), a) == 0
    return [tuple(a[1 + 3 * i:4 + 3 * i]) for i in range(a[0])]
