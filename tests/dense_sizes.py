"""Sizes (tokens, hidden, vocabulary or inner, type) that take, with those of test_gpu_dense.py, every form of launch of the
dense operators: product, tile, layout, result, planes, K parts, one launch or two (tests/test_dense_calls.py asserts it)."""
from silentotithrandousha_amd import MOE_BF16, MOE_F32

# loss and both gradients
LOSS = [(1, 32, 16448, MOE_F32), (1, 32, 32820, MOE_F32), (1, 2400, 193, MOE_BF16),
        (1, 2528, 193, MOE_BF16), (1, 2784, 165, MOE_F32), (1, 2880, 161, MOE_F32), (2, 2656, 323, MOE_BF16),
        (3, 2784, 162, MOE_BF16), (6, 32, 1, MOE_F32), (6, 32, 16458, MOE_F32), (11, 32, 33170, MOE_F32),
        (17, 32, 14929, MOE_BF16), (166, 2816, 1, MOE_BF16), (289, 1696, 1, MOE_BF16), (3273, 32, 131, MOE_BF16),
        (4094, 32, 35, MOE_BF16), (8031, 832, 5471, MOE_F32), (8195, 64, 9172, MOE_F32), (8279, 2880, 167, MOE_BF16),
        (8317, 832, 620, MOE_BF16), (8322, 32, 67, MOE_F32), (8669, 160, 38580, MOE_BF16), (9038, 1696, 33330, MOE_BF16),
        (9892, 1056, 43887, MOE_BF16), (10363, 96, 33935, MOE_BF16), (10939, 448, 35046, MOE_BF16),
        (11501, 544, 24617, MOE_BF16)]
# the gradient of the rows alone
LOSS_DX = [(1, 32, 24621, MOE_F32), (8211, 64, 7993, MOE_F32),
           (9017, 2112, 33080, MOE_BF16), (13715, 160, 5434, MOE_F32)]
# block, forward and backward
BLOCK = [(1, 32, 1544, MOE_F32), (1, 1504, 104, MOE_BF16), (1, 1536, 104, MOE_F32),
         (1, 2752, 56, MOE_F32), (1, 2752, 56, MOE_BF16), (3, 928, 4120, MOE_F32), (3, 2208, 4232, MOE_F32),
         (4, 32, 5320, MOE_F32), (4, 928, 2096, MOE_F32), (11, 2880, 1016, MOE_F32), (17, 1152, 3080, MOE_BF16),
         (33, 32, 4104, MOE_BF16), (33, 544, 6552, MOE_F32), (65, 32, 5448, MOE_F32), (66, 32, 3984, MOE_BF16),
         (187, 544, 7952, MOE_F32), (193, 2880, 4600, MOE_F32), (201, 2368, 40, MOE_BF16), (858, 768, 24, MOE_F32),
         (1080, 160, 3416, MOE_F32), (2336, 32, 704, MOE_F32), (2728, 1632, 6496, MOE_BF16), (7238, 288, 4864, MOE_BF16),
         (8341, 928, 8, MOE_BF16), (10513, 224, 1520, MOE_F32)]
# the same from a checkpoint
KEPT = [(1, 32, 1032, MOE_F32), (1, 32, 1032, MOE_BF16), (1, 32, 1544, MOE_BF16),
        (7, 2816, 4904, MOE_F32), (34, 2752, 8, MOE_BF16), (36, 1568, 1056, MOE_F32), (161, 2880, 8, MOE_BF16),
        (1217, 2880, 1608, MOE_BF16), (2724, 160, 7720, MOE_BF16), (4670, 288, 7944, MOE_BF16), (12300, 32, 8, MOE_BF16),
        (13278, 800, 8, MOE_BF16)]
