"""Sizes that reach each way the grouped products run, for the tests of the kernels (test_expert_tiles_gpu.py) and of the plan that
chooses among the ways (test_expert_plan_cpu.py)."""


def offsets_of(head, lengths):
    o = [head]
    for n in lengths:
        o.append(o[-1] + n)
    return o


# row counts of the experts: whole and part-filled tiles of 256 rows, ends below and above half a tile, one row, none; 15 tiles in all
LENGTHS = [700, 0, 1, 384, 1000, 129, 257, 500]

# 256 x 256 tiles in the forward product, the input gradient or both: name -> (rows, offsets, n, k, coarse in (NT, NN), tiles of the
# row range (rows of no expert included) left for the quarters of a second launch, of the larger of both tile counts)
COARSE = {
    'whole_rounds': (3008, offsets_of(0, LENGTHS), 4096, 4096, (True, True), 0),
    'few_left': (3028, offsets_of(20, LENGTHS), 4096, 4096, (True, True), 16),
    'a_quarter_left': (3871, offsets_of(300, LENGTHS), 4096, 4096, (True, True), 64),
    'a_last_round_of_whole_tiles': (4171, offsets_of(600, LENGTHS), 4096, 4096, (True, True), 80),
    'quarters_alone': (1000, offsets_of(0, [0] * 12 + [1000] + [0] * 11), 4096, 4096, (True, True), 64),
    'one_part_filled_round': (1030, offsets_of(0, [0] * 12 + [1000] + [0] * 11), 4096, 4096, (True, True), 80),
    'one_expert': (4200, offsets_of(0, [4200]), 4096, 4096, (True, True), 16),
    'padded_reduction_forward': (3028, offsets_of(20, LENGTHS), 4096, 4100, (True, False), 16),
    'part_filled_step_forward': (3028, offsets_of(20, LENGTHS), 4096, 4104, (True, False), 16),
    'padded_reduction_input_gradient': (3028, offsets_of(20, LENGTHS), 4100, 4096, (False, True), 16),
    'more_experts_than_lanes': (3100, offsets_of(40, [0, 90, 1] * 23 + [640]), 4096, 4096, (True, True), None),
}

# 128 x 128 tiles (32 x 128 where rows are few), results in 16-byte stores, several of them per workgroup:
# name -> (rows, offsets, n, k, least number of tiles of a workgroup in (NT, NN))
SEVERAL = {
    'one_step_forward': (40000, offsets_of(0, [9000, 0, 1, 15999, 130, 127, 4743, 10000]), 1024, 64, (3, 1)),
    'part_filled_steps_forward': (40000, offsets_of(30, [9000, 0, 1, 15999, 130, 127, 4743, 9900]), 1024, 136, (3, 1)),
    'one_step_input_gradient': (40000, offsets_of(0, [9000, 0, 1, 15999, 130, 127, 4743, 10000]), 64, 1024, (1, 3)),
    'part_filled_steps_input_gradient': (40000, offsets_of(30, [9000, 0, 1, 15999, 130, 127, 4743, 9900]), 200, 1024, (1, 3)),
    'tiles_of_32_rows': (2560, offsets_of(0, [40, 0, 33, 1, 86, 64, 32, 64] * 8), 2048, 2048, (2, 2)),
    'tiles_of_32_rows_more_experts_than_lanes': (3200, offsets_of(3, [40, 0, 33, 1, 86, 64, 32, 64] * 9 + [200]), 2048, 1024, (2, 1)),
}

# weight gradients: name -> (rows, offsets, n, k, whole experts as units, least number of tiles of a workgroup)
WEIGHT = {
    'whole_experts': (5000, offsets_of(0, [700, 0, 1, 384, 1000, 700, 257, 1900]), 2048, 1024, True, 2),
    'whole_experts_ragged': (5000, offsets_of(10, [700, 0, 1, 384, 1000, 700, 257, 1900]), 2040, 1096, True, 2),
    'whole_experts_equal': (2048, offsets_of(0, [256] * 8), 2048, 2048, True, 4),
    'cut_experts': (40000, offsets_of(0, [9000, 0, 1, 15999, 130, 127, 4743, 10000]), 520, 264, False, 1),
}

# 4-bit products: name -> (rows, offsets or None (dense), n, k, least number of tiles of a workgroup, slices of the reduction)
MX4 = {
    'one_step': (20000, offsets_of(0, [9000, 0, 1, 5870, 130, 127, 4872]), 1024, 256, 2, 1),
    'part_filled_steps': (20000, offsets_of(30, [9000, 0, 1, 5870, 130, 127, 4772]), 1024, 300, 2, 1),
    'three_steps': (20000, offsets_of(30, [9000, 0, 1, 5870, 130, 127, 4772]), 1152, 700, 2, 1),
    'dense': (20000, None, 1024, 96, 2, 1),
    'tiles_of_32_rows': (2560, offsets_of(0, [40, 0, 33, 1, 86, 64, 32, 64] * 8), 2048, 512, 2, 1),
    'sliced': (300, offsets_of(0, [100, 0, 150, 30]), 384, 4096, 1, 4),
    'sliced_dense': (200, None, 388, 2100, 1, 2),
    'sliced_rows_of_16_bytes': (700, offsets_of(3, [600, 90]), 256, 2048, 1, 2),
}

# 4-bit products of few rows per expert: name -> (rows, offsets, n, k, one launch for bf16, for float32 rows)
FEW = {
    'a_token': (1, offsets_of(0, [0, 1, 0]), 2048, 512, True, True),
    'sixteen_rows': (16, offsets_of(0, [1] * 7 + [0, 9]), 4096, 1024, True, True),
    'few_columns': (1000, offsets_of(0, [0, 30, 1, 16, 17] * 12 + [0, 200, 20, 0]), 64, 64, True, True),
    'by_the_type': (64, offsets_of(0, [0, 17, 1, 16, 9, 13, 8, 0]), 4096, 1024, True, False),
    'many_tiles': (256, offsets_of(0, [0, 17, 1, 16, 9, 13, 8, 0, 60, 20, 20, 33, 31, 1, 0, 27]), 2048, 512, True, True),
    'one_experts_rows': (1000, offsets_of(0, [0] * 5 + [1000] + [0] * 58), 2048, 512, False, False),
    'every_experts_rows': (1000, offsets_of(3, [0, 30, 1, 16, 17] * 12 + [0, 200, 20, 0]), 2048, 512, False, False),
}
