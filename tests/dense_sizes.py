"""Sizes at which dense layers and the loss on top of one take each of their forms: (inputs, outputs or channels, frames) and the form, as tests/cpp/test_dense_forms prints it.  test_dense_forms.py
holds the rules to it, test_gpu_dense_sizes.py runs them."""

FORWARD = {
    (20, 30, 8): "few",
    (300, 200, 40): "straight waves 8 slabs 1",
    (2048, 40, 70): "straight waves 8 slabs 8",
    (300, 2600, 2500): "packed small slabs 1 narrow",
    (1103, 640, 1300): "packed small slabs 4 narrow",
    (145, 21806, 548): "packed middle slabs 1 narrow",
    (8300, 700, 1100): "packed small slabs 8 wide",          # rows longer than the packing threads hold
}

# (the weights' gradient and the input's; wide: frames or outputs beyond what the packing threads hold)
BACKWARD = {
    (64, 64, 1030): "straight waves 8 slabs 3 and waves 8 slabs 1",
    (992, 579, 681): "packed small slabs 1 narrow and slabs 1",
    (700, 600, 1200): "packed small slabs 4 narrow and slabs 2",
    (4897, 1036, 1833): "packed middle slabs 1 narrow and slabs 1",
    (5000, 644, 814): "packed large slabs 1 narrow and slabs 1",
    (300, 2600, 1100): "packed large slabs 5 narrow and slabs 12",
    (600, 700, 8300): "packed large slabs 12 wide and slabs 1",
    (700, 8300, 600): "packed small slabs 1 wide and slabs 12",
}

# (more than 64 Mi logits: pieces, the last one shorter and no multiple of 32)
LOSS = {
    (24, 701, 100000): "straight pieces 2 last 189",
    (128, 701, 100000): "packed pieces 2 last 189 logits large slabs 1",
    (80, 9001, 9000): "packed pieces 2 last 1577 logits large slabs 1",
    (131, 3097, 4890): "packed pieces 1 last 3097 logits middle slabs 1",
    (470, 1378, 1260): "packed pieces 1 last 1378 logits small slabs 1",
    (2000, 700, 700): "packed pieces 1 last 700 logits small slabs 6",
}
