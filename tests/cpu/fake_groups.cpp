// Stands in for the embedded code object of the grouped products beside the model of the HIP runtime (fake_hip.cpp).
extern "C" {
extern const unsigned char maize_embedded_groups[1] = {0};
}
