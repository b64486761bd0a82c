"""Sizes (rows, inner, outer) at which the linear layer is tested."""

SIZES = [(1, 1, 1), (5, 3, 2), (1, 64, 256), (8, 256, 1000), (64, 32, 32), (257, 45, 100), (130, 64, 256), (300, 5, 32),
         (300, 32, 3), (77, 130, 40), (65, 256, 64), (33, 250, 1100), (2500, 16, 24), (1, 1100, 7), (40, 1000, 200),
         (3, 2000, 31), (513, 129, 33), (700, 600, 130)]

# each number of blocks of the contraction for which the weights stay in LDS, in
# 16-bit types and in float32, a slice of the columns and several; more rows than the
# kernel for few takes
RESIDENT = [(132000, 20, 5), (44000, 50, 70), (27000, 90, 129), (66000, 120, 64), (14000, 150, 300), (66007, 180, 33),
            (33000, 210, 100), (7000, 256, 610), (131500, 16, 1), (66000, 96, 40), (132000, 112, 8)]
# weights streamed: each number of column blocks of a slice
STREAMED = [(132000, 257, 20), (66000, 300, 50), (22000, 1000, 96), (33000, 333, 120), (27000, 270, 160), (11000, 520, 190),
            (9500, 1000, 200), (17000, 264, 256), (14000, 290, 290), (66000, 600, 3)]
# the others around which few rows' kernel ends, where every pair of types is tried
FEW = [(1025, 257, 20), (1100, 300, 50), (1300, 50, 70), (1500, 150, 300)]
# weight gradients that one workgroup holds (each of its shapes), rows from less than
# a block to several a workgroup
ONE_PASS = [(7, 64, 256), (33, 60, 250), (2100, 33, 200), (9000, 64, 96), (500, 128, 256), (4500, 70, 130), (40, 256, 64),
            (3000, 250, 50), (700, 256, 128), (5000, 129, 65), (20000, 8, 3)]
# float32 inputs in three blocks of the contraction: resident weights, one slice and several
THREE_BLOCKS = [(132000, 45, 5), (44000, 33, 70), (33000, 48, 129), (7000, 45, 1100)]
# gradients whose dx is a product with streamed weights
STREAMED_DX = [(rows, outer, inner) for rows, inner, outer in STREAMED]
