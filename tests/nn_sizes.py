"""Sizes at which the learned-head operators are tested in the mean square."""
# rows, dim, hidden
FFN_FEW = [(1, 1, 1), (5, 3, 2), (64, 32, 32), (257, 45, 100), (300, 96, 250), (77, 130, 40), (65, 256, 64),
           (33, 250, 1100), (1, 64, 5000), (40, 143, 946), (30, 70, 3), (4100, 20, 700), (100, 128, 96)]
# weights through LDS, whole or block by block
FFN_MANY = [(16500, 5, 9), (17001, 32, 600), (20011, 45, 100), (16399, 64, 1000), (9007, 96, 64), (8707, 128, 96),
            (8300, 200, 333), (8201, 256, 40), (65543, 200, 72), (131079, 112, 33)]
FFN_ALL = FFN_FEW + FFN_MANY
