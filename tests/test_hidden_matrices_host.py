"""Which parameters of the networks take Muon's transition."""


def test_head_rows_tables_and_vectors_stay_with_adamw():
    from pbg_b200 import postflop, preflop
    from pbg_b200.model_train import is_hidden_matrix

    for module in (preflop, postflop):
        shapes = module.parameter_shapes(preflop.PreflopConfig(), 13)
        hidden = {n for n, s in shapes.items() if is_hidden_matrix(n, s)}
        assert not any("embedding" in n or n.endswith(".bias") or "theta" in n for n in hidden)
        heads = {n for n in shapes if "_head." in n and n.endswith("affine.weight")}
        assert {"type_head.affine.weight", "raise_head.mixture_affine.weight"} <= heads and not heads & hidden
        assert {"value_head.features.w1.weight", "value_head.features.w2.weight", "attentions.0.w_qkv.weight"} <= hidden
