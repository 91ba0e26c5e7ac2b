"""Programs that use the library as a whole."""
