"""A weight image of the engine's layout with random values: enough to run the
engine where the published weights are not at hand."""
import json

import numpy as np


def tensor_shapes():
    shapes = {"features.embeddings.linear.weight": (16, 66),
              "features.embeddings.linear.bias": (16,),
              "features.edge_embedding.weight": (128, 416),
              "features.norm_edges.weight": (128,), "features.norm_edges.bias": (128,),
              "W_e.weight": (128, 128), "W_e.bias": (128,), "W_s.weight": (21, 128),
              "W_out.weight": (21, 128), "W_out.bias": (21,)}
    for part, wide, square, norms in (
            ("encoder_layers", {"W1": 384, "W11": 384}, ("W2", "W3", "W12", "W13"), 3),
            ("decoder_layers", {"W1": 512}, ("W2", "W3"), 2)):
        for layer in range(3):
            p = f"{part}.{layer}."
            for name, width in wide.items():
                shapes[p + name + ".weight"] = (128, width)
                shapes[p + name + ".bias"] = (128,)
            for name in square:
                shapes[p + name + ".weight"] = (128, 128)
                shapes[p + name + ".bias"] = (128,)
            for n in range(1, norms + 1):
                shapes[p + f"norm{n}.weight"] = (128,)
                shapes[p + f"norm{n}.bias"] = (128,)
            shapes[p + "dense.W_in.weight"] = (512, 128)
            shapes[p + "dense.W_in.bias"] = (512,)
            shapes[p + "dense.W_out.weight"] = (128, 512)
            shapes[p + "dense.W_out.bias"] = (128,)
    return shapes


def random_weights(seed=0) -> bytes:
    rng = np.random.default_rng(seed)
    header, data, at = {}, [], 0
    for name, shape in tensor_shapes().items():
        if "norm" in name and name.endswith("weight"):
            x = np.ones(shape)
        elif len(shape) == 2:
            x = rng.standard_normal(shape) / np.sqrt(shape[1])
        else:
            x = 0.1 * rng.standard_normal(shape)
        if name == "W_out.weight":
            x = 3.0 * x  # logits that spread like a trained model's
        raw = x.astype("<f4").tobytes()
        header[name] = {"dtype": "F32", "shape": list(shape), "data_offsets": [at, at + len(raw)]}
        data.append(raw)
        at += len(raw)
    text = json.dumps(header).encode()
    return len(text).to_bytes(8, "little") + text + b"".join(data)
